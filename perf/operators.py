"""What the operators between the projections of a decoder layer are measured on: the residual norm
(`add_rmsnorm`), the append to the 4-bit paged cache (`kv4_append`, read back with `kv4_read`) and the attention
over that cache (`kv4_attention`). `run` computes them in plain torch, or with `own` through the package."""

import math
import os
import random
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
EPS = 1e-5
TILE = 16  # tokens whose codes and scales are stored together


def _package():
    path = os.path.join(ROOT, "5090-blackwell-kernels_b200", "python")
    if path not in sys.path:
        sys.path.insert(0, path)
    import spark_kernels

    return spark_kernels


# ---- cases ----------------------------------------------------------------------------------------

def _norm(rows, hidden, post, gate, scale, **kw):
    return dict(op="norm", rows=rows, hidden=hidden, post=post, gate=gate, scale=scale, **kw)


def _append(seqs, q, ragged, len_max, hq, hkv, d, group, page, rot, **kw):
    return dict(op="append", seqs=seqs, q=q, ragged=ragged, len_max=len_max, hq=hq, hkv=hkv, d=d, group=group, page=page, rot=rot, **kw)


def _attention(seqs, q, ragged, len_max, hq, hkv, d, group, page, window, **kw):
    return dict(op="attention", seqs=seqs, q=q, ragged=ragged, len_max=len_max, hq=hq, hkv=hkv, d=d, group=group, page=page, window=window, **kw)


def listed():
    return [
        # one token of one sequence between attention and MLP: latency
        _norm(1, 4096, False, "none", 1.0, name="norm decode 1"),
        # a ragged prompt through a block with norms on both sides and a gate per channel
        _norm(4093, 5120, True, "channel", 1.0, name="norm both gate 4093"),
        # a long prompt batch, a gate for each token, scaled residual
        _norm(16384, 4096, True, "row", 0.7071, name="norm both rowgate 16384"),
        # a decode step of a small batch
        _append(16, 1, True, 2048, 32, 8, 128, 64, 64, 128, name="append decode 16"),
        # prompt chunks of different lengths, half of the channels rotated, other head shape
        _append(7, 1111, True, 3000, 20, 20, 64, 32, 16, 32, name="append chunks 7"),
        # one long prompt
        _append(1, 8192, False, 8192, 32, 8, 128, 64, 64, 128, name="append prompt 8192"),
        # a chat's first tokens: latency
        _attention(1, 1, False, 200, 32, 8, 128, 64, 64, 0, name="attend decode 1x200"),
        # a serving batch of mixed lengths, one slot empty
        _attention(64, 1, True, 4096, 32, 8, 128, 64, 64, 0, name="attend decode 64x4k"),
        # few sequences, long documents
        _attention(8, 1, False, 65536, 32, 8, 128, 128, 64, 0, name="attend decode 8x64k"),
        # every head its own keys, short pages, a window
        _attention(32, 1, True, 8000, 16, 16, 64, 32, 16, 1024, name="attend window 32x8k"),
        # verification of a few proposed tokens a sequence
        _attention(16, 5, True, 6001, 32, 8, 128, 64, 64, 0, name="attend verify 16x6k"),
        # a prompt chunk on top of a filled cache
        _attention(2, 2048, False, 8192, 32, 8, 128, 64, 64, 0, name="attend prompt 2x2k/8k"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "append", "attention", "attention"])
    if op == "norm":
        hidden = 8 * _log(rng, 64, 1024)
        rows = _log(rng, 1, min(16384, 16384 * 4096 // hidden))
        return _norm(rows, hidden, rng.random() < 0.5, rng.choice(["none", "channel", "row"]), rng.choice([1.0, 0.5, 1.25]))
    d = rng.choice([64, 128, 128])
    group = rng.choice([g for g in (32, 64, 128) if g <= d])
    hkv = rng.choice([1, 2, 4, 8])
    hq = hkv * rng.choice([1, 2, 4, 5, 7, 8, 16])
    page = rng.choice([16, 32, 64, 128])
    ragged = rng.random() < 0.7
    kind = rng.choice(["decode", "decode", "few", "prompt"])
    if op == "append":
        rot = rng.choice([d, d, d // 2])
        if kind == "decode":
            return _append(_log(rng, 1, 256), 1, ragged, _log(rng, 16, 8192), hq, hkv, d, group, page, rot)
        if kind == "few":
            q = rng.randint(2, 9)
            return _append(_log(rng, 1, 64), q, ragged, q + _log(rng, 16, 4000), hq, hkv, d, group, page, rot)
        q = _log(rng, 30, 4096)
        return _append(rng.randint(1, 2), q, ragged, q + _log(rng, 1, 3000), hq, hkv, d, group, page, rot)
    window = rng.choice([0, 0, 0, 128, 1000])
    if kind == "decode":
        seqs = _log(rng, 1, 128)
        return _attention(seqs, 1, ragged, _log(rng, 1, min(60000, 400000 // seqs)), hq, hkv, d, group, page, window)
    if kind == "few":
        seqs, q = _log(rng, 1, 32), rng.randint(2, 9)
        return _attention(seqs, q, ragged, q + _log(rng, 1, 60000 // seqs), hq, hkv, d, group, page, window)
    q = _log(rng, 30, 1500)
    return _attention(rng.randint(1, 2), q, ragged, q + _log(rng, 1, 5000), hkv * rng.choice([1, 4, 8]), hkv, d, group, page, window)


def _lengths(case):
    """New tokens and total length of every sequence: the case's alone, the same for every seed. The last sequence is a
    full one; of a ragged batch of single tokens with four sequences or more, the second is an empty slot."""
    rng = random.Random("%d %d %d %d" % (case["seqs"], case["q"], case["len_max"], case["hkv"]))
    n, lens = [], []
    for i in range(case["seqs"]):
        whole = not case["ragged"] or i == case["seqs"] - 1
        q = case["q"] if whole else rng.randint(max(1, case["q"] // 4), case["q"])
        n.append(q)
        lens.append(case["len_max"] if whole else rng.randint(q, case["len_max"]))
    if case["ragged"] and case["q"] == 1 and case["seqs"] >= 4:
        lens[1] = 0
    return n, lens


def _token_bytes(case):
    """Bytes of the cache for K and V of one token and head: the codes, and a scale and a minimum for each group."""
    return case["d"] + 8 * case["d"] // case["group"]


def work(case):
    if case["op"] == "norm":
        n = case["rows"] * case["hidden"]
        gate = {"none": 0, "channel": case["hidden"], "row": n}[case["gate"]]
        return {"bytes": 2 * (4 * n + gate + case["hidden"] * (2 if case["post"] else 1)), "flops": n * (8 if case["post"] else 5)}
    n, lens = _lengths(case)
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    if case["op"] == "append":
        t = sum(min(a, b) for a, b in zip(n, lens))
        moved = 2 * t * (hq + 2 * hkv) * d + 4 * t * case["rot"] + 2 * t * hq * d + t * hkv * _token_bytes(case)
        return {"bytes": moved + t * hkv * _token_bytes(case) + 4 * t * hkv * d, "flops": t * (3 * (hq + hkv) * case["rot"] + 8 * 2 * hkv * d)}
    w = case["window"]
    pairs = read = 0
    for q, length in zip(n, lens):
        first = length - q  # position of the first new token
        visible = [min(p + 1, w) if w else p + 1 for p in range(max(0, first), length)]
        pairs += sum(visible)
        read += length - (max(0, first - w + 1) if w else 0)
    return {"bytes": read * hkv * _token_bytes(case) + 4 * sum(n) * hq * d, "flops": 4 * pairs * hq * d}


# ---- inputs ---------------------------------------------------------------------------------------

def _pages(case, lens):
    """A page table [seqs, most pages] of pages in a shuffled order, and the number of pages in the pool."""
    per = max(1, -(-case["len_max"] // case["page"]))
    total = case["seqs"] * per + 3
    order = list(range(total))
    random.Random(total).shuffle(order)
    return torch.tensor(order[: case["seqs"] * per], dtype=torch.int32, device="cuda").reshape(case["seqs"], per), total


def _pack(kc, vc, ks, vs):
    """Codes uint8 [n, 16, d] and (minimum, scale) bf16 [n, 16, groups, 2] of K and V -> the bytes of n tiles.
    K: a token's row is four runs of d / 8 bytes, run c holding channels 32 i + 8 c .. + 7 for i = 0, 1, ...; V: blocks of
    eight tokens, in them eight runs g of eight tokens, a token's piece holding channels 32 u + 4 g .. + 3 for u = 0, 1, ...;
    the lower channel of a byte in its low bits. Then the words (minimum low, scale high) of K and of V."""
    n, t, d = kc.shape
    kb = kc.reshape(n, t, d // 32, 4, 4, 2)
    kb = (kb[..., 0] | kb[..., 1] << 4).permute(0, 1, 3, 2, 4).reshape(n, -1)
    vb = vc.reshape(n, 2, 8, d // 32, 8, 2, 2)
    vb = (vb[..., 0] | vb[..., 1] << 4).permute(0, 1, 4, 2, 3, 5).reshape(n, -1)
    return torch.cat([kb, vb, ks.reshape(n, -1).view(torch.uint8), vs.reshape(n, -1).view(torch.uint8)], 1)


def _unpack(tiles, d, group):
    """The inverse of `_pack`: float32 codes [n, 16, d] and the minima and scales [n, 16, groups] of K and V."""
    n, half, words = tiles.shape[0], TILE * d // 2, TILE * (d // group) * 4
    kb, vb, ks, vs = tiles.split([half, half, words, words], 1)
    kb = kb.reshape(n, TILE, 4, d // 32, 4).permute(0, 1, 3, 2, 4)
    vb = vb.reshape(n, 2, 8, 8, d // 32, 2).permute(0, 1, 3, 4, 2, 5)
    kc = torch.stack([kb & 15, kb >> 4], -1).reshape(n, TILE, d)
    vc = torch.stack([vb & 15, vb >> 4], -1).reshape(n, TILE, d)
    ks, vs = (x.contiguous().view(torch.bfloat16).reshape(n, TILE, d // group, 2) for x in (ks, vs))
    return kc, vc, ks, vs


def _codes(gen, shape):
    return torch.randn(shape, device="cuda", generator=gen).mul_(2.7).add_(7.5).round_().clamp_(0, 15).to(torch.uint8)


def _scales(gen, shape):
    """(minimum, scale) pairs of groups whose values are about normal, a few of them shifted."""
    s = torch.exp(0.3 * torch.randn(shape, device="cuda", generator=gen) - 1.1)
    m = -7.5 * s + 0.3 * torch.randn(shape, device="cuda", generator=gen)
    return torch.stack([m, s], -1).to(torch.bfloat16)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, device="cuda", generator=gen).to(torch.bfloat16)

    if case["op"] == "norm":
        h, rows = case["hidden"], case["rows"]
        gain = (1 + 0.1 * normal(2, h)).to(torch.bfloat16)
        gate = {"none": None, "channel": normal(h) if case["gate"] == "channel" else None,
                "row": normal(rows, h) if case["gate"] == "row" else None}[case["gate"]]
        return {"case": case, "x": 3 * normal(rows, h), "y": normal(rows, h), "gain": gain[0], "post": gain[1] if case["post"] else None, "gate": gate}
    n, lens = _lengths(case)
    hq, hkv, d, group = case["hq"], case["hkv"], case["d"], case["group"]
    table, total = _pages(case, lens)
    st = {"case": case, "table": table, "lens": torch.tensor(lens, dtype=torch.int32, device="cuda")}
    starts = [0]
    for q in n:
        starts.append(starts[-1] + q)
    st["offsets"] = None if case["q"] == 1 else torch.tensor(starts, dtype=torch.int32, device="cuda")
    seq = torch.repeat_interleave(torch.arange(len(n), device="cuda"), torch.tensor(n, device="cuda"))
    pos = torch.arange(starts[-1], device="cuda") - torch.tensor(starts, device="cuda")[seq] + (torch.tensor(lens, device="cuda") - torch.tensor(n, device="cuda"))[seq]
    tiles = case["page"] // TILE
    tile_bytes = TILE * _token_bytes(case)
    if case["op"] == "append":
        # the projection's output, keys with a few loud channels; the rotation's table of a common base
        qkv = normal(starts[-1], (hq + 2 * hkv) * d)
        qkv[:, hq * d: (hq + hkv) * d: 37] *= 6
        inv = 500000.0 ** (-torch.arange(0, case["rot"], 2, device="cuda", dtype=torch.float64) / case["rot"])
        ang = torch.arange(case["len_max"], device="cuda", dtype=torch.float64)[:, None] * inv
        st["table_cs"] = torch.cat([ang.cos(), ang.sin()], 1).float()
        slots = table[seq, pos.clamp(min=0) // case["page"]].long() * case["page"] + pos.clamp(min=0) % case["page"]
        st |= {"qkv": qkv, "pos": pos, "slots": torch.where(pos >= 0, slots, -1),
               "pool": torch.zeros(total, hkv, tiles, tile_bytes, dtype=torch.uint8, device="cuda")}
        return st
    count = total * hkv * tiles
    pool = torch.empty(count, tile_bytes, dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 26) // (TILE * d))
    for a in range(0, count, step):
        b = min(count, a + step)
        pool[a:b] = _pack(_codes(gen, (b - a, TILE, d)), _codes(gen, (b - a, TILE, d)), _scales(gen, (b - a, TILE, d // group)), _scales(gen, (b - a, TILE, d // group)))
    pool = pool.reshape(total, hkv, tiles, tile_bytes)
    # what lies behind the last token of a sequence was never written: any bytes, NaN among them
    for b, length in enumerate(lens):
        first = -(-length // TILE)
        flat = table[b].long().repeat_interleave(tiles) * tiles + torch.arange(tiles, device="cuda").repeat(table.shape[1])
        pool.view(total, hkv, tiles, tile_bytes)[flat[first:] // tiles, :, flat[first:] % tiles] = 255
    q = 1.5 * normal(starts[-1], hq, d)
    return st | {"pool": pool, "q": q, "seq": seq, "pos": pos, "tokens": n}


# ---- the plain forms --------------------------------------------------------------------------------

def _norm_plain(st):
    case, x, y = st["case"], st["x"].float(), st["y"].float()
    if st["post"] is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * st["post"].float()
    if st["gate"] is not None:
        y = y * st["gate"].float()
    r = (case["scale"] * x + y).to(torch.bfloat16)
    f = r.float()
    return r, (f * torch.rsqrt((f * f).mean(-1, keepdim=True) + EPS) * st["gain"].float()).to(torch.bfloat16)


def _rotate(x, cs):
    """x [t, heads, d], cs [t, rot] (cosines, sines): the two halves of the first rot channels rotated."""
    half = cs.shape[1] // 2
    c, s = cs[:, None, :half], cs[:, None, half:]
    a, b = x[..., :half], x[..., half: 2 * half]
    return torch.cat([a * c - b * s, b * c + a * s, x[..., 2 * half:]], -1)


def _four_bits(x, group):
    """The values that x's codes of 4 bits stand for, group by group."""
    g = x.reshape(*x.shape[:-1], -1, group)
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    m = lo.to(torch.bfloat16).to(x.dtype)
    s = ((hi - m) / 15).clamp(min=0).to(torch.bfloat16).to(x.dtype)
    s = torch.where(s < 2.0 ** -126, torch.zeros_like(s), s)
    c = torch.where(s > 0, torch.round((g - m) / s), torch.zeros_like(g)).clamp(0, 15)  # a division: halves lie on the border
    return (c * s + m).reshape(x.shape)


def _append_parts(st, cast):
    case, t = st["case"], st["qkv"].shape[0]
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    q, k, v = st["qkv"].to(cast).split([hq * d, hkv * d, hkv * d], 1)
    real = (st["pos"] >= 0)[:, None, None]
    cs = st["table_cs"][st["pos"].clamp(min=0)].to(cast)
    return q.reshape(t, hq, d), k.reshape(t, hkv, d), v.reshape(t, hkv, d), cs, real


def _append_plain(st):
    q, k, v, cs, real = _append_parts(st, torch.float32)
    g = st["case"]["group"]
    zero = torch.zeros((), device="cuda")
    q = torch.where(real, _rotate(q, cs), zero)
    k = torch.where(real, _four_bits(_rotate(k, cs), g), zero)
    v = torch.where(real, _four_bits(v, g), zero)
    return q.to(torch.bfloat16), k.to(torch.bfloat16), v.to(torch.bfloat16)


def _dequantized(tiles, d, group, cast):
    kc, vc, ks, vs = _unpack(tiles, d, group)

    def value(c, ms):
        ms = ms.to(cast)
        return (c.to(cast).reshape(*c.shape[:2], -1, group) * ms[..., 1:] + ms[..., :1]).reshape(c.shape)

    return value(kc, ks), value(vc, vs)


def _attention_plain(st):
    case = st["case"]
    b, hq, hkv, d = case["seqs"], case["hq"], case["hkv"], case["d"]
    tiles, most, rep = case["page"] // TILE, max(st["tokens"]), case["hq"] // case["hkv"]
    pages = st["pool"][st["table"].long()]                                     # [b, pages, hkv, tiles, bytes]
    k, v = _dequantized(pages.transpose(1, 2).reshape(-1, pages.shape[-1]), d, case["group"], torch.float32)
    length = pages.shape[1] * case["page"]
    j = torch.arange(length, device="cuda")
    held = (j < st["lens"][:, None])[:, None, :, None]
    zero = torch.zeros((), device="cuda")
    k = torch.where(held, k.reshape(b, hkv, length, d), zero)
    v = torch.where(held, v.reshape(b, hkv, length, d), zero)
    # queries padded to the most tokens of a sequence: [b, hkv, most * rep, d]
    starts = torch.searchsorted(st["seq"], torch.arange(b, device="cuda"))
    place = torch.arange(st["q"].shape[0], device="cuda") - starts[st["seq"]]
    q = torch.zeros(b, most, hq, d, device="cuda")
    q[st["seq"], place] = st["q"].float()
    pos = torch.full((b, most), -1, device="cuda")
    pos[st["seq"], place] = st["pos"]
    seen = j <= pos[..., None]
    if case["window"]:
        seen &= j > pos[..., None] - case["window"]
    bias = torch.where(seen, zero, torch.full((), float("-inf"), device="cuda"))
    q = q.reshape(b, most, hkv, rep, d).permute(0, 2, 1, 3, 4).reshape(b, hkv, most * rep, d)
    s = torch.matmul(q, k.transpose(-1, -2)).mul_(1 / math.sqrt(d))
    s = s.reshape(b, hkv, most, rep, length).add_(bias[:, None, :, None, :])
    top = s.amax(-1, keepdim=True)
    p = s.sub_(torch.where(top > float("-inf"), top, zero)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.reshape(b, hkv, most * rep, length), v).reshape(b, hkv, most, rep, d)
    o = torch.where(total > 0, o / total, zero).permute(0, 2, 1, 3, 4).reshape(b, most, hq, d)
    return o[st["seq"], place].to(torch.bfloat16)


def run(state):
    case = state["case"]
    if case["op"] == "norm":
        if own:
            return _package().add_rmsnorm(state["x"], state["y"], state["gain"], eps=EPS, post_gain=state["post"], gate=state["gate"], residual_scale=case["scale"])
        return _norm_plain(state)
    if case["op"] == "append":
        if own:
            sk = _package()
            cache = sk.KV4Cache.from_pool(state["pool"], case["d"], case["group"])
            q = sk.kv4_append(state["qkv"], cache, state["table"], state["lens"], state["table_cs"], q_offsets=state["offsets"])
            return (q, *sk.kv4_read(cache, state["slots"]))
        return _append_plain(state)
    if own:
        sk = _package()
        cache = sk.KV4Cache.from_pool(state["pool"], case["d"], case["group"])
        return sk.kv4_attention(state["q"], cache, state["table"], state["lens"], q_offsets=state["offsets"], window=case["window"])
    return _attention_plain(state)


# ---- in 64 bits ---------------------------------------------------------------------------------------

def _values64(tiles, d, group):
    """K and V of tiles as float64 [tokens, d], every channel's byte looked up on its own."""
    ch, t = torch.arange(d, device="cuda"), torch.arange(TILE, device="cuda")[:, None]
    low, words = 4 * (ch % 2), TILE * d
    kat = t * (d // 2) + ch % 32 // 8 * (d // 8) + ch // 32 * 4 + ch % 8 // 2
    vat = TILE * d // 2 + t // 8 * 4 * d + ch % 32 // 4 * (d // 2) + t % 8 * (d // 16) + ch // 32 * 2 + ch % 4 // 2
    out = []
    for at, base in ((kat, words), (vat, words + TILE * (d // group) * 4)):
        word = base + (t * (d // group) + ch // group) * 4

        def half(offset):
            bits = tiles[:, word + offset].to(torch.int32) | tiles[:, word + offset + 1].to(torch.int32) << 8
            return (bits << 16).view(torch.float32).double()

        out.append(((tiles[:, at] >> low & 15).double() * half(2) + half(0)).reshape(-1, d))
    return out


def exact(case, seed):
    st = prepare(case, seed)
    f = torch.float64
    if case["op"] == "norm":
        x, z = st["x"].to(f), st["y"].to(f)
        if st["post"] is not None:
            z = z / ((z ** 2).sum(-1, keepdim=True) / case["hidden"] + EPS).sqrt() * st["post"].to(f)
        r = case["scale"] * x + (z if st["gate"] is None else z * st["gate"].to(f))
        held = r.to(torch.bfloat16).to(f)  # the next norm is of the residual as it is stored
        return r, held / ((held ** 2).sum(-1, keepdim=True) / case["hidden"] + EPS).sqrt() * st["gain"].to(f)
    if case["op"] == "append":
        q, k, v, cs, real = _append_parts(st, f)
        c, s = cs[:, None].chunk(2, -1)
        half = c.shape[-1]

        def turned(x):
            y = x.clone()
            y[..., :half] = x[..., :half] * c - x[..., half: 2 * half] * s
            y[..., half: 2 * half] = x[..., half: 2 * half] * c + x[..., :half] * s
            return y

        def coded(x):
            g = x.unflatten(-1, (-1, case["group"]))
            m = g.min(-1, keepdim=True).values.to(torch.bfloat16).to(f)
            w = ((g.max(-1, keepdim=True).values - m) / 15).to(torch.bfloat16).to(f)
            return (((g - m) / w).round().clamp(0, 15) * w + m).flatten(-2)

        return tuple(x * real for x in (turned(q), coded(turned(k)), coded(v)))
    rep, d, out, at = case["hq"] // case["hkv"], case["d"], [], 0
    for b, count in enumerate(st["tokens"]):
        length = int(st["lens"][b])
        q = st["q"][at: at + count].to(f)
        pos = st["pos"][at: at + count]
        at += count
        if length == 0:
            out.append(torch.zeros_like(q))
            continue
        pages = st["pool"][st["table"][b, : -(-length // case["page"])].long()]
        heads = []
        for h in range(case["hkv"]):
            k, v = (x[:length] for x in _values64(pages[:, h].reshape(-1, pages.shape[-1]), d, case["group"]))
            j = torch.arange(length, device="cuda")
            hidden = j[None] > pos[:, None]
            if case["window"]:
                hidden |= j[None] <= pos[:, None] - case["window"]
            for i in range(rep):
                s = (q[:, h * rep + i] @ k.T) / d ** 0.5
                heads.append(torch.softmax(s.masked_fill(hidden, float("-inf")), -1) @ v)
        out.append(torch.stack(heads, 1))
    return torch.cat(out)
