"""A decode step of a Llama-style decoder on the quantized projections of this library: the caller side
of the path, in the order the reference's engine runs it (python/spark_kernels/engine.py:441-456,
`_layers_quant`): per layer
    rmsnorm -> qkv projection -> rope + KV-cache append -> attention over the cache -> o projection ->
    residual add + rmsnorm -> gate|up projection -> SwiGLU -> down projection -> residual add
and its replay from a CUDA graph (engine.py:870-899). The four projections are `quant.make_linear`
objects (int4, fp8, mxfp8, nvfp4 ...), or, for int4 with `fuse_swiglu`, the fused gate|up + SwiGLU GEMM
of this library. What lies between them comes in two forms. With the default bf16 cache, plain torch stands in for the
reference's row kernels, and the module is about the data flow through the projections (every GEMM consumes
the previous one's output, unlike a benchmark over fixed buffers). With kv="int4" the step runs on this library's
operators from end to end: `add_rmsnorm` (residual and norm in one launch), `kv4_append` (rotation and a 4-bit
paged cache) and `kv4_attention`; `extend` then also takes several tokens of a sequence at once, e.g. its prompt.

`TorchDecoder` is the same arithmetic on the dequantized weights in bf16 torch matmuls, which is what the
reference checks its engine against (tests/test_quant.py:94-105).
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from . import kv4
from . import ops as sk
from . import quant

KV_PAGE = 64  # tokens of a page of the 4-bit cache


@dataclass(frozen=True)
class DecoderConfig:
    hidden: int = 4096
    q_heads: int = 32
    kv_heads: int = 8
    head_dim: int = 128
    intermediate: int = 14336
    layers: int = 32
    rope_theta: float = 500000.0
    eps: float = 1e-5

    @property
    def qkv_cols(self) -> int:
        return (self.q_heads + 2 * self.kv_heads) * self.head_dim


def random_weights(cfg: DecoderConfig, device, seed: int = 0) -> list[dict]:
    """bf16 weights of `cfg.layers` layers, [in, out] as the Linear classes take them: wqkv, wo, w_gate_up
    (gate columns first, then up), w_down, and the two norm gains."""
    g = torch.Generator(device=device).manual_seed(seed)
    h, inter = cfg.hidden, cfg.intermediate

    def w(k, n):
        return (torch.randn(k, n, device=device, generator=g) / k ** 0.5).to(torch.bfloat16)

    return [{"wqkv": w(h, cfg.qkv_cols), "wo": w(cfg.q_heads * cfg.head_dim, h), "w_gate_up": w(h, 2 * inter), "w_down": w(inter, h),
             "norm1": (1 + 0.1 * torch.randn(h, device=device, generator=g)).to(torch.bfloat16),
             "norm2": (1 + 0.1 * torch.randn(h, device=device, generator=g)).to(torch.bfloat16)} for _ in range(cfg.layers)]


def rmsnorm(x: torch.Tensor, gain: torch.Tensor, eps: float) -> torch.Tensor:
    xf = x.float()
    return (xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps) * gain.float()).to(torch.bfloat16)


def rope(x: torch.Tensor, pos: torch.Tensor, theta: float) -> torch.Tensor:
    """x [B, heads, d], pos [B]: rotate the two halves of every head by pos * theta^(-2 i / d)."""
    d = x.shape[-1]
    inv = theta ** (-torch.arange(0, d, 2, device=x.device, dtype=torch.float32) / d)
    ang = pos.float()[:, None, None] * inv
    cos, sin = ang.cos(), ang.sin()
    x1, x2 = x.float()[..., : d // 2], x.float()[..., d // 2:]
    return torch.cat([x1 * cos - x2 * sin, x2 * cos + x1 * sin], -1).to(torch.bfloat16)


class _Projections:
    """The four projections of one layer as callables."""

    def __init__(self, w: dict, fmt: str, fuse_swiglu: bool):
        self.qkv, self.o, self.down = (quant.make_linear(w[k], fmt) for k in ("wqkv", "wo", "w_down"))
        self.fused = fuse_swiglu and fmt in ("int4", "int4-asym")
        if self.fused:
            self.gate_up_w = sk.W4GateUpWeight.quantize(w["w_gate_up"], asym=fmt == "int4-asym")
        else:
            self.gate_up = quant.make_linear(w["w_gate_up"], fmt)

    def mlp_in(self, h: torch.Tensor) -> torch.Tensor:
        """silu(gate) * up of the gate|up projection: one fused launch, or GEMM + torch."""
        if self.fused:
            return sk.w4gemm_swiglu(h, self.gate_up_w)
        gu = self.gate_up(h)
        inter = gu.shape[1] // 2
        return (torch.nn.functional.silu(gu[:, :inter].float()) * gu[:, inter:].float()).to(torch.bfloat16)


class _Dense:
    """bf16 torch matmul on a given [K, N] weight (the comparison model's projections)."""

    def __init__(self, w: torch.Tensor):
        self.w = w

    def __call__(self, a: torch.Tensor) -> torch.Tensor:
        return a @ self.w


class QuantizedDecoder:
    """Decoder whose projections run on this library. `decode(x, pos)` advances every sequence of the batch by
    one token: x [B, hidden] bf16 are the embedded tokens, pos [B] int64 their positions; the KV cache holds
    `max_len` positions per sequence, in bf16, or with kv="int4" in 4 bits (head_dim 64 or 128). A position at or past max_len is
    an error: the bf16 cache fails at the index; the 4-bit one leaves the token out of the cache, so that row's result means
    nothing, and `_C.device_status()` returns 5 (a captured step cannot raise: ask after the steps whose lengths may have ended)."""

    def __init__(self, cfg: DecoderConfig, weights: list[dict], fmt: str = "int4", fuse_swiglu: bool = True,
                 batch: int = 1, max_len: int = 64, kv: str = "bf16"):
        if kv not in ("bf16", "int4"):
            raise ValueError(f"unknown cache format {kv!r}; expected 'bf16' or 'int4'")
        self.cfg, self.fmt = cfg, fmt
        dev = weights[0]["wqkv"].device
        self.layers = [self._projections(w, fmt, fuse_swiglu) for w in weights]
        self.norms = [(w["norm1"], w["norm2"]) for w in weights]
        self.kv = kv
        if kv == "int4":
            # every sequence has the pages for max_len tokens; a serving engine would hand them out as sequences grow
            per = -(-max_len // KV_PAGE)
            self.cache = [kv4.KV4Cache(batch * per, cfg.kv_heads, cfg.head_dim, KV_PAGE, min(64, cfg.head_dim), device=dev) for _ in weights]
            self.page_table = torch.arange(batch * per, dtype=torch.int32, device=dev).reshape(batch, per)
            self.cos_sin = kv4.rotation_table(max_len, cfg.head_dim, cfg.rope_theta, device=dev)
        else:
            shape = (cfg.layers, batch, cfg.kv_heads, max_len, cfg.head_dim)
            self.k_cache = torch.zeros(shape, dtype=torch.bfloat16, device=dev)
            self.v_cache = torch.zeros(shape, dtype=torch.bfloat16, device=dev)
        self.device = dev
        self.max_len = max_len
        self._graph = None

    def _projections(self, w, fmt, fuse_swiglu):
        return _Projections(w, fmt, fuse_swiglu)

    def dequantized_weights(self) -> list[dict]:
        """The weights the quantized projections really multiply by, for the comparison model."""
        out = []
        for lay, (n1, n2) in zip(self.layers, self.norms):
            if lay.fused:
                # undo the strip interleave: dequantize, then put gate strips first and up strips second
                full = quant.formats.w4_dequantize(lay.gate_up_w.packed, lay.gate_up_w.scales, lay.gate_up_w.zeros)
                strips = full.reshape(full.shape[0], -1, 16)
                gate_up = torch.cat([strips[:, 0::2].reshape(full.shape[0], -1), strips[:, 1::2].reshape(full.shape[0], -1)], 1)
            else:
                gate_up = lay.gate_up.dequantize()
            out.append({"wqkv": lay.qkv.dequantize(), "wo": lay.o.dequantize(), "w_gate_up": gate_up,
                        "w_down": lay.down.dequantize(), "norm1": n1, "norm2": n2})
        return out

    def decode(self, x: torch.Tensor, pos: torch.Tensor) -> torch.Tensor:
        cfg = self.cfg
        if self.kv == "int4":
            return self.extend(x, (pos + 1).to(torch.int32))
        B = x.shape[0]
        rows = torch.arange(B, device=x.device)
        # keys at positions <= pos are visible; the mask is computed from pos on the device (graph safe)
        visible = torch.arange(self.max_len, device=x.device)[None, :] <= pos[:, None]
        bias = torch.zeros(B, 1, 1, self.max_len, dtype=torch.float32, device=x.device).masked_fill(~visible[:, None, None, :], float("-inf"))
        for li, (lay, (n1, n2)) in enumerate(zip(self.layers, self.norms)):
            h = rmsnorm(x, n1, cfg.eps)
            qkv = lay.qkv(h)
            q, k, v = qkv.split([cfg.q_heads * cfg.head_dim, cfg.kv_heads * cfg.head_dim, cfg.kv_heads * cfg.head_dim], -1)
            q = rope(q.reshape(B, cfg.q_heads, cfg.head_dim), pos, cfg.rope_theta)
            k = rope(k.reshape(B, cfg.kv_heads, cfg.head_dim), pos, cfg.rope_theta)
            self.k_cache[li, rows, :, pos] = k
            self.v_cache[li, rows, :, pos] = v.reshape(B, cfg.kv_heads, cfg.head_dim)
            rep = cfg.q_heads // cfg.kv_heads
            keys = self.k_cache[li].repeat_interleave(rep, 1).float()   # [B, q_heads, L, d]
            vals = self.v_cache[li].repeat_interleave(rep, 1).float()
            att = torch.softmax((q.float()[:, :, None, :] @ keys.transpose(-1, -2)) / cfg.head_dim ** 0.5 + bias, -1) @ vals
            x = x + lay.o(att.reshape(B, -1).to(torch.bfloat16))
            x = x + lay.down(lay.mlp_in(rmsnorm(x, n2, cfg.eps)))
        return x

    def extend(self, x: torch.Tensor, lens: torch.Tensor, q_offsets: torch.Tensor | None = None) -> torch.Tensor:
        """kv="int4" only: the hidden states after the last layer for the new tokens x [rows, hidden] of the sequences.
        lens int32 [n], n at most `batch`: tokens of the first n sequences after this call (0: an empty slot); q_offsets int32
        [n + 1]: rows q_offsets[b] .. q_offsets[b + 1] - 1 are the new tokens of sequence b, its last ones; None: one each."""
        if self.kv != "int4":
            raise ValueError("extend needs kv='int4'")
        table = self.page_table[: lens.shape[0]]
        r, h = sk.add_rmsnorm(x, gain=self.norms[0][0], eps=self.cfg.eps)
        for li, lay in enumerate(self.layers):
            q = kv4.kv4_append(lay.qkv(h), self.cache[li], table, lens, self.cos_sin, q_offsets)
            att = kv4.kv4_attention(q, self.cache[li], table, lens, q_offsets)
            r, h = sk.add_rmsnorm(r, lay.o(att.reshape(x.shape[0], -1)), gain=self.norms[li][1], eps=self.cfg.eps)
            nxt = self.norms[li + 1][0] if li + 1 < len(self.layers) else None
            r, h = sk.add_rmsnorm(r, lay.down(lay.mlp_in(h)), gain=nxt, eps=self.cfg.eps)
        return r

    # ---- CUDA-graph replay of the step (fixed buffers, as the reference's engine does) ----
    def capture(self, batch: int) -> None:
        dev = self.device
        self._x = torch.zeros(batch, self.cfg.hidden, dtype=torch.bfloat16, device=dev)
        self._pos = torch.zeros(batch, dtype=torch.int64, device=dev)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):  # warm-up: every scratch of the library exists before capture
            self.decode(self._x, self._pos)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        if self.kv == "int4":
            for c in self.cache:
                c.pool.zero_()
        else:
            self.k_cache.zero_()
            self.v_cache.zero_()
        self._graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self._graph):
            self._y = self.decode(self._x, self._pos)

    def replay(self, x: torch.Tensor, pos: torch.Tensor) -> torch.Tensor:
        self._x.copy_(x)
        self._pos.copy_(pos)
        self._graph.replay()
        return self._y


class TorchDecoder(QuantizedDecoder):
    """The comparison model: the same step with bf16 torch matmuls on given (dequantized) weights."""

    def __init__(self, cfg: DecoderConfig, weights: list[dict], batch: int = 1, max_len: int = 64):
        super().__init__(cfg, weights, fmt="dense", fuse_swiglu=False, batch=batch, max_len=max_len)

    def _projections(self, w, fmt, fuse_swiglu):
        class P:
            fused = False
            qkv, o, gate_up, down = _Dense(w["wqkv"]), _Dense(w["wo"]), _Dense(w["w_gate_up"]), _Dense(w["w_down"])
            mlp_in = _Projections.mlp_in
        return P()
