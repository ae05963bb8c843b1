"""The operators over the 4-bit KV cache and the residual norm in 64 bits, in plain torch on the CPU, and the sizes
their tests share. Written from the definitions in include/spk.h and the byte layout in csrc/kv4_layout.cuh."""

import torch

F64 = torch.float64


def unpack(pool: torch.Tensor, d: int, group: int):
    """pool uint8 [pages, heads, tiles, bytes] -> K and V as float64 [pages, tiles * 16, heads, d]."""
    pages, heads, tiles, _ = pool.shape
    flat = pool.cpu().reshape(pages * heads * tiles, -1)
    n = flat.shape[0]
    out = []
    for which in range(2):
        codes = torch.zeros(n, 16, d, dtype=torch.int64)
        for t in range(16):
            for ch in range(d):
                if which == 0:
                    byte = t * (d // 2) + ch % 32 // 8 * (d // 8) + ch // 32 * 4 + ch % 8 // 2
                else:
                    byte = 8 * d + t // 8 * 4 * d + ch % 32 // 4 * (d // 2) + t % 8 * (d // 16) + ch // 32 * 2 + ch % 4 // 2
                codes[:, t, ch] = flat[:, byte].long() >> 4 * (ch % 2) & 15
        at = 16 * d + which * 64 * (d // group)
        words = flat[:, at: at + 64 * (d // group)].contiguous().view(torch.bfloat16).reshape(n, 16, d // group, 2).to(F64)
        v = codes.to(F64) * words[..., 1].repeat_interleave(group, -1) + words[..., 0].repeat_interleave(group, -1)
        out.append(v.reshape(pages, heads, tiles * 16, d).transpose(1, 2))
    return out


def rotate(x: torch.Tensor, cs: torch.Tensor) -> torch.Tensor:
    """x [t, heads, d] float64, cs [t, rot] float32."""
    rot = cs.shape[1]
    c, s = cs[:, None, : rot // 2].to(F64), cs[:, None, rot // 2:].to(F64)
    a, b = x[..., : rot // 2], x[..., rot // 2: rot]
    return torch.cat([a * c - b * s, b * c + a * s, x[..., rot:]], -1)


def quantize(x: torch.Tensor, group: int):
    """x [..., d] float64 -> (values, scales, minima) of its codes, [..., d] each."""
    g = x.unflatten(-1, (-1, group))
    m = g.amin(-1, keepdim=True).to(torch.bfloat16).to(F64)
    s = ((g.amax(-1, keepdim=True) - m).float() * (1 / 15)).clamp(min=0).to(torch.bfloat16).to(F64)  # in fp32, as defined
    s = torch.where(s < 2.0 ** -126, torch.zeros_like(s), s)
    c = torch.where(s > 0, ((g - m) / s).round().clamp(0, 15), torch.zeros_like(g))
    return (c * s + m).flatten(-2), s.expand_as(g).flatten(-2), m.expand_as(g).flatten(-2)


def rows_of(lens, q_offsets):
    """(sequence, position) of every row that belongs to a sequence."""
    out = []
    for b, length in enumerate(lens):
        n = 1 if q_offsets is None else q_offsets[b + 1] - q_offsets[b]
        out += [(b, length - n + i) for i in range(n)]
    return out


def attention(q, k, v, table, lens, q_offsets, scale, window):
    """q [rows, hq, d]; k, v [pages, page, hkv, d] float64; -> float64 [rows, hq, d] and, per row and head, the bound of what
    the kernel may be off by: sums below."""
    q = q.cpu().to(F64)
    hq, hkv, page = q.shape[1], k.shape[2], k.shape[1]
    out, slack = torch.zeros_like(q), torch.zeros_like(q)
    for row, (b, pos) in enumerate(rows_of(lens, q_offsets)):
        lo = max(0, pos - window + 1) if window else 0
        if pos < 0:
            continue
        j = torch.arange(lo, pos + 1)
        pages, at = torch.tensor(table[b])[j // page], j % page
        for h in range(hq):
            kk, vv = k[pages, at, h * hkv // hq], v[pages, at, h * hkv // hq]
            out[row, h] = torch.softmax(kk @ q[row, h] * scale, -1) @ vv
            slack[row, h] = vv.abs().amax(0)
    return out, slack
