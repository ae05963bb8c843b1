"""A paged KV cache in 4 bits and the operators over it: `kv4_append` (rotate q and k, quantize k and v into the
cache), `kv4_attention` (attention over the cache) and `kv4_read` (the values of named tokens). An addition to the
reference's surface, whose cache is bf16.

Every call over the cache is told what its sequences are by the same arguments, all int32 on the device, so that a
captured CUDA graph serves growing sequences:

    lens [seqs]               tokens of each sequence in the cache, this call's included
    page_table [seqs, width]  the pages of each sequence, in order
    q_offsets [seqs + 1]      this call's rows of sequence b are q_offsets[b] .. q_offsets[b + 1] - 1, its last
                              tokens; None: one row per sequence (a decode step)

Row i of n of a sequence has position lens - n + i; a row of negative position (an empty slot of a padded batch) is
padding: it is not appended, and its q and its attention output are zeros. Pages may be shared between sequences for
reading; two sequences of one call must not append to the same page. Indices are checked on the device: a page
outside the pool or a position outside the rotation's table is left out, the rows of a sequence whose length is past
its row of the table are padding, and each makes `_C.device_status()` return 5. Forward only.
"""

from __future__ import annotations

import torch

from . import _C


class KV4Cache:
    """Keys and values of one layer in 4 bits: `pages` pages of `page_size` tokens for `kv_heads` heads, each `group`
    channels of a token with a bf16 scale and minimum of their own. head_dim 64 or 128; group 32, 64 or 128, at most
    head_dim; page_size a multiple of 16 up to 1024. A token costs head_dim + 8 head_dim / group bytes a head, K and V
    together (bf16: 4 head_dim)."""

    def __init__(self, pages: int, kv_heads: int, head_dim: int = 128, page_size: int = 64, group: int = 64, device="cuda"):
        nbytes = _C.kv4_tile_bytes(head_dim, group)
        if nbytes == 0:
            raise ValueError(f"KV4Cache supports head_dim 64 or 128 and group 32, 64 or 128 (at most head_dim), got head_dim={head_dim} group={group}")
        if page_size % 16 or not 16 <= page_size <= 1024 or pages < 1 or kv_heads < 1:
            raise ValueError(f"KV4Cache needs page_size a multiple of 16 up to 1024, pages and kv_heads at least 1, got {page_size}, {pages}, {kv_heads}")
        self._set(torch.zeros(pages, kv_heads, page_size // 16, nbytes, dtype=torch.uint8, device=device), head_dim, group)

    def _set(self, pool: torch.Tensor, head_dim: int, group: int) -> None:
        self.pool, self.head_dim, self.group = pool, head_dim, group

    @staticmethod
    def from_pool(pool: torch.Tensor, head_dim: int = 128, group: int = 64) -> "KV4Cache":
        """A cache over existing memory: uint8 [pages, kv_heads, page_size / 16, kv4_tile_bytes(head_dim, group)], e.g.
        a layer's part of one allocation for all layers."""
        _C._check_pool(pool, head_dim, group, "KV4Cache")
        cache = KV4Cache.__new__(KV4Cache)
        cache._set(pool, head_dim, group)
        return cache

    @property
    def pages(self) -> int:
        return self.pool.shape[0]

    @property
    def kv_heads(self) -> int:
        return self.pool.shape[1]

    @property
    def page_size(self) -> int:
        return 16 * self.pool.shape[2]

    def nbytes(self) -> int:
        return self.pool.numel()


def kv4_append(qkv: torch.Tensor, cache: KV4Cache, page_table: torch.Tensor, lens: torch.Tensor, cos_sin: torch.Tensor | None,
               q_offsets: torch.Tensor | None = None, q_out: torch.Tensor | None = None) -> torch.Tensor:
    """qkv [rows, (Hq + 2 Hkv) head_dim] bf16 (the projection's output; rows may be strided): q and k rotated by their
    positions, k and v quantized into the cache, q returned as bf16 [rows, Hq, head_dim]. cos_sin float32
    [positions, rot]: cosines then sines of the rotation of the first rot channels, whose halves are the pairs
    (rot a multiple of 8; None: no rotation). Per group of the (unrounded) channels y: m = bf16(min y),
    s = bf16((max y - m) * (1 / 15)) in fp32, code = clamp(rint((y - m) / s), 0, 15), value = code * s + m; a group that holds an
    infinity or a NaN reads back as NaN. Rows of a given q_out behind the last sequence are left as they were (zeros
    in one that the call allocates)."""
    return _C.kv4_append(qkv, cache.pool, page_table, lens, cos_sin, q_offsets, cache.head_dim, cache.group, q_out)


def kv4_attention(q: torch.Tensor, cache: KV4Cache, page_table: torch.Tensor, lens: torch.Tensor, q_offsets: torch.Tensor | None = None,
                  scale: float | None = None, window: int = 0, out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of q [rows, Hq, head_dim] bf16 over the cache: every row sees the positions up to its own, with
    window > 0 the last `window` of them; softmax of scale * q.k (default head_dim ** -0.5) in fp32, bf16 out
    [rows, Hq, head_dim]. Hq is a multiple of the cache's heads, query head h reading head h // (Hq // Hkv). A row that
    sees nothing gets zeros. Rows of a given `out` behind the last sequence are left as they were (zeros in one that
    the call allocates); `out` must not lie in q's memory. The weighted values are summed in fp32 before they are
    divided by the weights' sum: values of up to 1e27 are safe at every length. Weights are rounded to fp16, 2^-11 of each and
    2^-28 of the row's largest (times its group's scale); in prompts values are too, to 2^-11 and 2^-32 of the largest before
    them in any group, and a weight of a token whose values are more than 2^16 below the loudest loses a bit for each 2 past that."""
    return _C.kv4_attention(q, cache.pool, page_table, lens, q_offsets, cache.head_dim, cache.group,
                            cache.head_dim ** -0.5 if scale is None else scale, window, out)


def kv4_read(cache: KV4Cache, slots: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Keys (rotated) and values of the tokens in `slots` (int64 [n], page * page_size + place in the page) as bf16
    [n, Hkv, head_dim] each; zeros for a negative slot."""
    return _C.kv4_read(cache.pool, slots, cache.head_dim, cache.group)


def rotation_table(positions: int, rot: int, theta: float = 10000.0, device="cuda") -> torch.Tensor:
    """float32 [positions, rot], cosines then sines of p * theta^(-2 i / rot): the table `kv4_append` takes. Angles in
    64 bits (in 32 those of far positions are off by more than the table's rounding)."""
    inv = theta ** (-torch.arange(0, rot, 2, device=device, dtype=torch.float64) / rot)
    ang = torch.arange(positions, device=device, dtype=torch.float64)[:, None] * inv
    return torch.cat([ang.cos(), ang.sin()], 1).float()
