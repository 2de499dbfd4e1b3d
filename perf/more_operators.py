"""The attention block of a decoder layer in 8 bits, as cases that can be timed and compared.

Four kinds of case:

  product  Int8Linear: rows quantised to 8 bits, each with a scale, times a matrix in 8 bits with a scale per channel
  rotate   HeadRope: biases, norms of queries and keys for each head and the rotation by position in one pass
  store    KvCache8.store, then KvCache8.load of every position of the blocks it wrote
  attend   KvCache8.attend: causal attention over the 8-bit cache, one new row a sequence (decode) or runs of rows

8 bits.  A group of values (a row of the product's activations, a row of its weights, a block of the cache) has the
scale s = max|v| / 127 and the codes round(v * (127 / max|v|)), halves to even; every step is rounded to 32 bits, and
what is held is s * code.

The cache.  A block is 16 positions of one kv head, its keys and its values with one scale each: `scales` f32
[page][kv head][page / 64 tiles][keys, values][4 blocks].  A tile is 64 positions of one kv head, 64 (qd + vd) bytes of
`codes`, [page][kv head][page / 64 tiles][keys, values]:

  keys    [block T of 4][qd / 16][position 16][16 bytes: the dims]
  values  [vd / 16][g 4][dim 16][block T of 4][i 4]: position 16 T + 4 g + i

The codes of a block that is not full yet are those of its positions so far; the values of the positions before the
rows written now are what an earlier store wrote.
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
        # One token through a square projection (o of a hidden size of 4096): the smallest call.
        {"name": "product_one", "kind": "product", "t": 1, "n": 4096, "k": 4096},
        # A decode step's q, k and v of 32 sequences in one product (32 heads over 8 of 128).
        {"name": "product_decode", "kind": "product", "t": 32, "n": 6144, "k": 4096},
        # A latent projection (512 + 64 channels) of a chunk, sizes off every tile.
        {"name": "product_odd", "kind": "product", "t": 333, "n": 576, "k": 2048},
        # The largest: a batch of prompts through q, k and v.
        {"name": "product_prompt", "kind": "product", "t": 8191, "n": 6144, "k": 4096},
        # A decode step's queries and keys, with a norm for each head.
        dict(_heads(GROUPED), name="rotate_decode", kind="rotate", rows=32, norm=True, bias=False, rot=128, far=4000),
        # Prompts far into long contexts.
        dict(_heads(GROUPED), name="rotate_prompt", kind="rotate", rows=16376, norm=True, bias=False, rot=128, far=100000),
        # A decode step's rows, blocks open at every filling.
        dict(_heads(GROUPED), name="store_decode", kind="store", seqs=32, new=1, past=1500, page=64),
        # The largest write: a batch of long prompts behind a shared beginning of odd length.
        dict(_heads(GROUPED), name="store_prompts", kind="store", seqs=8, new=2047, past=45, page=64),
        # Batched decode.
        dict(_heads(GROUPED), name="attend_decode", kind="attend", seqs=32, new=1, past=1500, page=64, window=0, pad=0),
        # One user far into a long context: the position axis is all the parallelism there is.
        dict(_heads(GROUPED), name="attend_one_long", kind="attend", seqs=1, new=1, past=100001, page=64, window=0,
             pad=0),
        # Chunks of four prompts of a latent-attention model; the launch is sized for more rows than there are.
        dict(_heads(LATENT), name="attend_chunks", kind="attend", seqs=4, new=61, past=3001, page=128, window=0, pad=4),
        # A long prompt.
        dict(_heads(GROUPED), name="attend_prompt", kind="attend", seqs=1, new=4001, past=0, page=64, window=0, pad=0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["product", "product", "rotate", "store", "attend", "attend", "attend"])
    if kind == "product":
        k = 16 * _log(rng, 4, 700)
        n = _log(rng, 16, 12000)
        return {"kind": "product", "t": _log(rng, 1, max(2, min(8000, 2 * 10 ** 11 // (n * k)))), "n": n, "k": k}
    h = rng.choice(HEADS)
    c = dict(_heads(h), kind=kind)
    if kind == "rotate":
        rot = rng.choice([h[2], h[2], h[2] // 2])
        c["norm"], c["bias"] = rng.random() < 0.7, rng.random() < 0.4
        return dict(c, rows=_log(rng, 1, 60000 // (h[0] + h[1])), rot=rot, far=_log(rng, 10, 200000))
    c["page"] = rng.choice([64, 64, 128, 256])
    if kind == "store":
        seqs = _log(rng, 1, 64)
        return dict(c, seqs=seqs, new=_log(rng, 1, 8000 // seqs), past=rng.randint(0, 1000))
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
    if c["kind"] == "product":
        t, n, k = c["t"], c["n"], c["k"]
        return {"bytes": 4 * t * k + n * k + 4 * n + 4 * t * n, "flops": 2 * t * n * k}
    h, kv, qd, vd = c["heads"], c["kv_heads"], c["qd"], c["vd"]
    if c["kind"] == "rotate":
        values = c["rows"] * (h + kv) * qd
        return {"bytes": 8 * values, "flops": 6 * values}
    new = c["new"]
    rows = c["seqs"] * new
    if c["kind"] == "store":
        # rows in, codes and scales out and in again, rows out; an open block's earlier rows come out again too
        again = sum(p % 16 for p in _pasts(c))
        return {"bytes": (rows * 4 + (rows + again) * (1 + 1 + 4)) * kv * (qd + vd), "flops": 0}
    w = c["window"]
    seen = sum(min(p + new, w + new - 1) if w else p + new for p in _pasts(c))
    pairs = sum(sum(min(p + i + 1, w) if w else p + i + 1 for i in range(new)) for p in _pasts(c))
    return {"bytes": 4 * rows * h * (qd + vd) + seen * kv * (qd + vd + 0.5), "flops": 2 * pairs * h * (qd + vd)}


# ------------------------------------------------------------------- inputs


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _prepare_product(c, seed):
    g = _gen(seed)
    t, n, k = c["t"], c["n"], c["k"]
    # Rows of differing size and a few channels far larger than the rest, as activations have them.
    x = torch.randn((t, k), generator=g, device=DEV) * torch.exp(torch.randn((t, 1), generator=g, device=DEV))
    x[:, torch.randint(0, k, (max(1, k // 500),), generator=g, device=DEV)] *= 8.0
    w = torch.randn((n, k), generator=g, device=DEV) * (0.02 + 0.02 * torch.rand((n, 1), generator=g, device=DEV))
    st = {"case": c, "x": x, "y": torch.empty((t, n), device=DEV)}
    if own:
        from moe_amd.int8 import Int8Linear

        st["own"] = Int8Linear(w)
    else:
        st["w"], st["w_scale"] = _quantise(w)  # a program has its weights quantised once
    return st


def _prepare_rotate(c, seed):
    g = _gen(seed)
    rows, h, kv, qd = c["rows"], c["heads"], c["kv_heads"], c["qd"]
    normal = lambda *s: torch.randn(s, generator=g, device=DEV)  # noqa: E731
    st = {"case": c, "q": normal(rows, h * qd) * 2.0, "k": normal(rows, kv * qd) * torch.exp(normal(rows, 1)),
          "pos": torch.randint(0, c["far"], (rows,), generator=g, device=DEV, dtype=torch.int32),
          "inv": (10000.0 ** (-torch.arange(0, c["rot"], 2, device=DEV, dtype=torch.float64) / c["rot"])).float()}
    for name, width in (("q", h * qd), ("k", kv * qd)):
        st[name + "_out"] = torch.empty_like(st[name])
        st[name + "_norm"] = 1.0 + 0.2 * normal(qd) if c["norm"] else None
        st[name + "_bias"] = 0.5 * normal(width) if c["bias"] else None
    if own:
        from moe_amd.heads import HeadRope

        st["own"] = HeadRope(h, kv, qd, st["inv"], dim=c["rot"], q_norm=st["q_norm"], k_norm=st["k_norm"],
                             q_bias=st["q_bias"], k_bias=st["k_bias"], eps=1e-6)
    return st


def _prepare_cache(c, g):
    """A table of scattered pages, and the new rows' sequences and positions."""
    P, new = c["page"], c["new"]
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
    pad = c.get("pad", 0)
    pos = torch.cat([torch.arange(p, p + new) for p in pasts] + [torch.full((pad,), -1)])
    seq = torch.cat([torch.full((new,), i) for i in range(n)] + [torch.zeros(pad, dtype=torch.int64)])
    return {"case": c, "table": table, "pages": n_pages, "pos": pos.to(DEV, torch.int32), "seq": seq.to(DEV, torch.int32),
            "max_pos": max(pasts) + new - 1}


def _slots(st, seq, pos):
    P = st["case"]["page"]
    return st["table"][seq.long(), (pos // P).long()].long() * P + pos % P


def _rows_of(st, seq, pos):
    """A step's rows as PageTable.advance would give them."""
    from moe_amd.paged import Rows

    n = st["case"]["seqs"]
    start = torch.searchsorted(seq.contiguous(), torch.arange(n + 1, device=DEV, dtype=torch.int32)).to(torch.int32)
    return Rows(start, seq, pos, _slots(st, seq, pos), torch.zeros(n, dtype=torch.int32, device=DEV))


def _prepare_store(c, seed):
    g = _gen(seed)
    st = _prepare_cache(c, g)
    kv, qd, vd, new = c["kv_heads"], c["qd"], c["vd"], c["new"]
    normal = lambda *s: torch.randn(s, generator=g, device=DEV)  # noqa: E731
    # Every position of the blocks the step touches: those of an earlier step first, then the new ones.
    pasts = _pasts(c)
    count = torch.tensor([p % 16 + new for p in pasts])
    seq = torch.repeat_interleave(torch.arange(len(pasts)), count)
    pos = torch.cat([torch.arange(p - p % 16, p + new) for p in pasts])
    fresh = torch.cat([torch.arange(p % 16 + new) >= p % 16 for p in pasts]).to(DEV)
    st["all_seq"], st["all_pos"], st["fresh"] = seq.to(DEV, torch.int32), pos.to(DEV, torch.int32), fresh
    rows = len(pos)
    # Keys and values of differing size, some rows far larger.
    big = torch.exp(normal(rows, 1))
    k, v = normal(rows, kv * qd) * big, normal(rows, kv * vd) * big
    st["k"], st["v"] = k[fresh].contiguous(), v[fresh].contiguous()
    st["old_k"], st["old_v"] = k[~fresh].contiguous(), v[~fresh].contiguous()
    st["k_out"], st["v_out"] = torch.empty_like(k), torch.empty_like(v)
    if own:
        from moe_amd.paged import KvCache8

        st["own"] = cache = KvCache8.new(st["pages"], st["table"], n_kv=kv, qd=qd, vd=vd, page=c["page"])
        old = ~fresh
        if len(st["old_k"]):
            cache.store(st["old_k"], st["old_v"], _rows_of(st, st["all_seq"][old], st["all_pos"][old]))
        st["rows"] = _rows_of(st, st["seq"], st["pos"])
        st["all_slots"] = _slots(st, st["all_seq"], st["all_pos"])
    return st


def _prepare_attend(c, seed):
    g = _gen(seed)
    st = _prepare_cache(c, g)
    kv, qd, vd, P = c["kv_heads"], c["qd"], c["vd"], c["page"]
    tiles = st["pages"] * kv * (P // 64)
    tb = 64 * (qd + vd)
    codes = torch.empty((tiles, tb), dtype=torch.int8, device=DEV)
    # Codes as N(0, 1) values get them (the largest of a block's 2000 at 127), scales as of values of that size.
    step = max(1, (1 << 27) // tb)
    for t in range(0, tiles, step):
        k = min(step, tiles - t)
        codes[t:t + k] = (torch.randn((k, tb), generator=g, device=DEV) * 37.0).round_().clamp_(-127, 127).to(torch.int8)
    st["codes"] = codes
    st["scales"] = torch.rand((tiles, 2, 4), generator=g, device=DEV) * 0.01 + 0.022
    # Queries sharp enough that some positions matter more than most.
    rows = len(st["pos"])
    st["q"] = torch.randn((rows, c["heads"] * qd), generator=g, device=DEV) * 2.0
    st["scale"] = qd ** -0.5
    st["out"] = torch.zeros((rows, c["heads"] * vd), device=DEV)
    if own:
        from moe_amd.paged import KvCache8

        b = KvCache8.sizes(st["pages"], c["seqs"], n_kv=kv, qd=qd, vd=vd, page=P)
        st["own"] = KvCache8(codes.view(torch.uint8).view(-1), st["scales"].view(-1),
                             torch.zeros(b[2], dtype=torch.uint8, device=DEV), st["table"], n_kv=kv, qd=qd, vd=vd, page=P)
    return st


def prepare(case, seed):
    c = dict(case)
    return {"product": _prepare_product, "rotate": _prepare_rotate, "store": _prepare_store,
            "attend": _prepare_attend}[c["kind"]](c, seed)


# ------------------------------------------------------------- the plain forms


def _quantise(x):
    """[groups, values] f32 -> codes f32, scales f32 [groups]."""
    top = x.abs().amax(-1)
    inv = torch.where(top > 0, (127.0 / top.double()).float(), torch.zeros_like(top))  # (rounded once, to 32 bits)
    return torch.round(x * inv[:, None]), (top.double() / 127.0).float()


def _plain_product(st):
    code, scale = _quantise(st["x"])
    st["y"].copy_(torch.matmul(code, st["w"].t()) * (scale[:, None] * st["w_scale"]))
    return [st["y"]]


def _plain_rotate(st):
    c = st["case"]
    rows, qd, rot = c["rows"], c["qd"], c["rot"]
    # The angle is the 32-bit product of position and frequency, as the models are trained with; far ones lose too
    # much in a 32-bit sine.
    angle = (st["pos"].float()[:, None] * st["inv"]).double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    for name in "qk":
        x = st[name] if st[name + "_bias"] is None else st[name] + st[name + "_bias"]
        x = x.view(rows, -1, qd)
        if st[name + "_norm"] is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * st[name + "_norm"]
        a, b = x[..., : rot // 2], x[..., rot // 2: rot]
        st[name + "_out"].copy_(torch.cat([a * cos - b * sin, a * sin + b * cos, x[..., rot:]], -1).view(rows, -1))
    return [st["q_out"], st["k_out"]]


def _plain_store(st):
    c = st["case"]
    kv, fresh = c["kv_heads"], st["fresh"]
    # Blocks in the order of the rows, and each row's.
    key = st["all_seq"].long() * (1 << 32) + st["all_pos"].long() // 16
    _, block = torch.unique_consecutive(key, return_inverse=True)
    n = sum((p % 16 + c["new"] + 15) // 16 for p in _pasts(c))
    for name, d in (("k", c["qd"]), ("v", c["vd"])):
        x = torch.empty_like(st[name + "_out"])
        x[fresh], x[~fresh] = st[name], st["old_" + name]
        full = torch.zeros((n, 16, kv, d), device=DEV)
        full[block, st["all_pos"].long() % 16] = x.view(-1, kv, d)
        code, scale = _quantise(full.transpose(1, 2).reshape(n * kv, 16 * d))
        held = (code * scale[:, None]).view(n, kv, 16, d)
        st[name + "_out"].copy_(held[block, :, st["all_pos"].long() % 16].reshape(-1, kv * d))
    return [st["k_out"], st["v_out"]]


def _cached(st, keys):
    """Every sequence's keys or values, [sequence, kv head, position, width] f32, from the tiles."""
    c = st["case"]
    n, kv, qd, vd, P = c["seqs"], c["kv_heads"], c["qd"], c["vd"], c["page"]
    page = st["table"][:, :-1].clamp(min=0).long()
    tiles = st["codes"].view(st["pages"], kv, P // 64, -1)[page].transpose(1, 2)  # [seq, kv, page, tile, bytes]
    scale = st["scales"].view(st["pages"], kv, P // 64, 2, 4)[page].transpose(1, 2)[..., 0 if keys else 1, :]
    if keys:
        x = tiles[..., :64 * qd].reshape(n, kv, -1, 4, qd // 16, 16, 16).transpose(-3, -2)  # [.., T, position, dims]
        x = x.reshape(n, kv, -1, 16, qd)
    else:
        x = tiles[..., 64 * qd:].reshape(n, kv, -1, vd // 16, 4, 16, 4, 4)  # [.., D, g, dim, T, i]
        x = x.permute(0, 1, 2, 6, 4, 7, 3, 5).reshape(n, kv, -1, 16, vd)
    return (x.float() * scale.reshape(n, kv, -1, 1, 1)).reshape(n, kv, -1, x.shape[-1])


def _plain_attend(st):
    c = st["case"]
    n, new, kv, qd, vd, h = (c[k] for k in ("seqs", "new", "kv_heads", "qd", "vd", "heads"))
    rep = h // kv
    kt = _cached(st, True).transpose(2, 3).contiguous()
    pos = st["pos"][: n * new].view(n, 1, 1, new, 1)
    q = st["q"][: n * new].view(n, new, kv, rep, qd).permute(0, 2, 3, 1, 4).reshape(n, kv, rep * new, qd)
    s = torch.matmul(q, kt) * st["scale"]
    del kt
    at = torch.arange(s.shape[-1], device=DEV)
    seen = at <= pos
    if c["window"]:
        seen = seen & (at > pos - c["window"])
    s = torch.where(seen, s.view(n, kv, rep, new, -1), -math.inf).view(n, kv, rep * new, -1)
    e = torch.exp(s - s.amax(-1, keepdim=True))
    del s
    o = torch.matmul(e, _cached(st, False)) / e.sum(-1, keepdim=True)
    st["out"][: n * new] = o.view(n, kv, rep, new, vd).permute(0, 3, 1, 2, 4).reshape(n * new, h * vd)
    return [st["out"]]


# ------------------------------------------------------------- the framework's


def _run_own(st):
    c, op = st["case"], st["own"]
    if c["kind"] == "product":
        op(st["x"], st["y"])
        return [st["y"]]
    if c["kind"] == "rotate":
        op(st["q"], st["k"], st["pos"], q_out=st["q_out"], k_out=st["k_out"])
        return [st["q_out"], st["k_out"]]
    if c["kind"] == "store":
        op.store(st["k"], st["v"], st["rows"])
        op.load(st["all_slots"], st["k_out"], st["v_out"])
        return [st["k_out"], st["v_out"]]
    op.attend(st["q"], st["seq"], st["pos"], st["out"], max_pos=st["max_pos"], scale=st["scale"], window=c["window"])
    return [st["out"]]


def run(state):
    if own:
        return _run_own(state)
    return {"product": _plain_product, "rotate": _plain_rotate, "store": _plain_store,
            "attend": _plain_attend}[state["case"]["kind"]](state)


# ------------------------------------------------------------------- 64 bits


def _exact_codes(x):
    """Codes and scales as they are defined, each step rounded to 32 bits (a product or quotient of two 32-bit numbers
    rounded once from 64 is that): max / 127, 127 / max, the value times it, the nearest whole number, even at halves."""
    top = x.double().abs().max(-1, keepdim=True).values
    inv = torch.where(top > 0, 127.0 / top, top).float().double()
    y = (x.double() * inv).float().double()
    low = torch.floor(y)
    odd = torch.remainder(low, 2.0)
    code = low + ((y - low > 0.5) | ((y - low == 0.5) & (odd == 1.0))).double()
    return code, (top / 127.0).float().double()


def _exact_tile_values(st, i, head, upto, keys):
    """Positions 0 .. upto - 1 of one sequence's kv head in 64 bits, byte by byte from the tiles."""
    c = st["case"]
    P, kv, qd, vd = c["page"], c["kv_heads"], c["qd"], c["vd"]
    d = qd if keys else vd
    p = torch.arange(upto, device=DEV)
    tile = (st["table"][i].long()[p // P] * kv + head) * (P // 64) + p % P // 64
    j = torch.arange(d, device=DEV)
    t = (p % 64)[:, None]
    if keys:
        byte = t // 16 * (16 * qd) + j // 16 * 256 + t % 16 * 16 + j % 16
    else:
        byte = 64 * qd + j // 16 * 1024 + t % 16 // 4 * 256 + j % 16 * 16 + t // 16 * 4 + t % 4
    code = st["codes"].view(-1)[tile[:, None] * (64 * (qd + vd)) + byte]
    scale = st["scales"].view(-1)[tile * 8 + (0 if keys else 4) + p % 64 // 16]
    return code.double() * scale.double()[:, None]


def exact(case, seed):
    global own
    c, mine = dict(case), own
    own = False  # inputs alone: no handle of the framework's
    try:
        st = prepare(c, seed)
        if c["kind"] == "product":
            # (made again rather than kept, in the order prepare makes them)
            g = _gen(seed)
            t, n, k = c["t"], c["n"], c["k"]
            torch.randn((t, k), generator=g, device=DEV), torch.randn((t, 1), generator=g, device=DEV)
            torch.randint(0, k, (max(1, k // 500),), generator=g, device=DEV)
            w = torch.randn((n, k), generator=g, device=DEV) * (0.02 + 0.02 * torch.rand((n, 1), generator=g, device=DEV))
    finally:
        own = mine
    if c["kind"] == "product":
        (x, sx), (w, sw) = _exact_codes(st["x"]), _exact_codes(w)
        return [torch.mm(x, w.t().contiguous()) * sx * sw.t()]
    if c["kind"] == "rotate":
        rows, qd, rot = c["rows"], c["qd"], c["rot"]
        angle = (st["pos"].double()[:, None] * st["inv"].double()).float().double()  # rounded to 32 bits by definition
        turn = torch.polar(torch.ones_like(angle), angle)[:, None]
        out = []
        for name in "qk":
            x = st[name].double()
            if c["bias"]:
                x = x + st[name + "_bias"].double()
            x = x.view(rows, -1, qd)
            if c["norm"]:
                x = st[name + "_norm"].double() * x / (x.square().sum(-1, keepdim=True) / qd + 1e-6).sqrt()
            z = torch.complex(x[..., : rot // 2].contiguous(), x[..., rot // 2: rot].contiguous()) * turn
            out.append(torch.cat([z.real, z.imag, x[..., rot:]], -1).view(rows, -1))
        return out
    if c["kind"] == "store":
        out = []
        for name, d in (("k", c["qd"]), ("v", c["vd"])):
            got, new, old, at = [], st[name].view(-1, c["kv_heads"], d), st["old_" + name].view(-1, c["kv_heads"], d), 0
            for i, past in enumerate(_pasts(c)):
                r = past % 16
                x = torch.cat([old[at:at + r], new[i * c["new"]:(i + 1) * c["new"]]])
                at += r
                pad = -len(x) % 16
                full = torch.cat([x, torch.zeros((pad, *x.shape[1:]), device=DEV)]).view(-1, 16, c["kv_heads"], d)
                code, scale = _exact_codes(full.permute(0, 2, 1, 3).reshape(-1, c["kv_heads"], 16 * d))
                held = (code * scale).view(-1, c["kv_heads"], 16, d).permute(0, 2, 1, 3).reshape(-1, c["kv_heads"] * d)
                got.append(held[: len(x)])
            out.append(torch.cat(got))
        return out
    n, new, h, kv, qd, vd, win = (c[k] for k in ("seqs", "new", "heads", "kv_heads", "qd", "vd", "window"))
    rep, pos = h // kv, st["pos"].long()
    out = torch.zeros((len(pos), h, vd), dtype=torch.float64, device=DEV)
    for i in range(n):
        upto = int(pos[(i + 1) * new - 1]) + 1
        at = torch.arange(upto, device=DEV)
        for g in range(kv):
            k, v = (_exact_tile_values(st, i, g, upto, keys) for keys in (True, False))
            # A sequence's rows at once where their scores fit.
            step = max(1, (1 << 28) // (rep * upto))
            for a in range(i * new, (i + 1) * new, step):
                b = min(a + step, (i + 1) * new)
                q = st["q"][a:b].view(b - a, h, qd)[:, g * rep:(g + 1) * rep].double()
                s = torch.mm(q.reshape(-1, qd), k.t().contiguous()).view(b - a, rep, upto) * float(st["scale"])
                top = pos[a:b, None, None]
                hide = at > top
                if win:
                    hide = hide | (at <= top - win)
                p = torch.softmax(s.masked_fill(hide, -math.inf), -1)
                out[a:b, g * rep:(g + 1) * rep] = torch.mm(p.view(-1, upto), v).view(b - a, rep, vd)
    return [out.view(len(pos), h * vd)]
