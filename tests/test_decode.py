"""A decode step through the quantized projections (python/spark_kernels/decode.py) against the same step
with bf16 torch matmuls on the dequantized weights, and its CUDA-graph replay against eager execution.
Mirrors the reference's whole-model checks (tests/test_quant.py:94-105,119-148): two layers, a few steps,
relative error of the hidden state per weight format (the comparison model does not quantize activations,
hence the wider bounds for the fp8 / fp4 formats)."""

import pytest
import torch

pytestmark = pytest.mark.gpu

TOL = {"int4": 2e-2, "int4-asym": 2e-2, "fp8-tok": 8e-2, "mxfp8": 8e-2, "nvfp4": 2.5e-1}


def _cfg(sk):
    from spark_kernels.decode import DecoderConfig

    return DecoderConfig(hidden=512, q_heads=4, kv_heads=2, head_dim=128, intermediate=1024, layers=2)


@pytest.mark.parametrize("fmt", list(TOL))
@pytest.mark.parametrize("batch", [1, 4])
def test_decode_steps_match_dense_model(sk, fmt, batch):
    from spark_kernels import decode

    cfg = _cfg(sk)
    w = decode.random_weights(cfg, "cuda", seed=5)
    q = decode.QuantizedDecoder(cfg, w, fmt=fmt, batch=batch, max_len=8)
    ref = decode.TorchDecoder(cfg, q.dequantized_weights(), batch=batch, max_len=8)
    g = torch.Generator(device="cuda").manual_seed(6)
    for step in range(3):
        x = torch.randn(batch, cfg.hidden, device="cuda", generator=g).to(torch.bfloat16)
        pos = torch.full((batch,), step, dtype=torch.int64, device="cuda")
        got, want = q.decode(x, pos).float(), ref.decode(x, pos).float()
        rel = ((got - want).norm() / want.norm()).item()
        assert rel < TOL[fmt], (fmt, batch, step, rel)
    assert sk._C.device_status() == 0


def test_fused_swiglu_and_two_step_mlp_agree(sk):
    from spark_kernels import decode

    cfg = _cfg(sk)
    w = decode.random_weights(cfg, "cuda", seed=7)
    a = decode.QuantizedDecoder(cfg, w, fmt="int4", fuse_swiglu=True, batch=2, max_len=4)
    b = decode.QuantizedDecoder(cfg, w, fmt="int4", fuse_swiglu=False, batch=2, max_len=4)
    x = torch.randn(2, cfg.hidden, device="cuda").to(torch.bfloat16)
    pos = torch.zeros(2, dtype=torch.int64, device="cuda")
    ya, yb = a.decode(x, pos).float(), b.decode(x, pos).float()
    assert ((ya - yb).norm() / yb.norm()).item() < 1e-2


def test_graph_replay_equals_eager(sk):
    """The step captured once and replayed (fixed buffers, positions read on the device) gives the eager bits."""
    from spark_kernels import decode

    cfg = _cfg(sk)
    w = decode.random_weights(cfg, "cuda", seed=8)
    eager = decode.QuantizedDecoder(cfg, w, fmt="int4", batch=2, max_len=8)
    graphed = decode.QuantizedDecoder(cfg, w, fmt="int4", batch=2, max_len=8)
    graphed.capture(2)
    g = torch.Generator(device="cuda").manual_seed(9)
    for step in range(4):
        x = torch.randn(2, cfg.hidden, device="cuda", generator=g).to(torch.bfloat16)
        pos = torch.full((2,), step, dtype=torch.int64, device="cuda")
        assert torch.equal(graphed.replay(x, pos), eager.decode(x, pos)), step


def _reference_step(decode, ref, cfg, weights, state, x, where):
    """A step over the 4-bit cache in plain torch: x [rows, hidden], where[row] = (sequence, position). Keys and values are
    rounded to what their 4-bit codes stand for; `state[layer][sequence]` is the list of (k, v) so far."""
    cs = torch.cat([f(torch.arange(64)[:, None] * cfg.rope_theta ** (-torch.arange(0, cfg.head_dim, 2, dtype=torch.float64) / cfg.head_dim)) for f in (torch.cos, torch.sin)], 1)
    pos = torch.tensor([p for _, p in where])
    for li, w in enumerate(weights):
        qkv = (decode.rmsnorm(x, w["norm1"], cfg.eps) @ w["wqkv"]).cpu().double().reshape(len(where), -1, cfg.head_dim)
        turned = ref.rotate(qkv[:, : cfg.q_heads + cfg.kv_heads], cs[pos])
        k = ref.quantize(turned[:, cfg.q_heads:], 64)[0]
        v = ref.quantize(qkv[:, cfg.q_heads + cfg.kv_heads:], 64)[0]
        for row, (b, _) in enumerate(where):
            state[li][b].append((k[row], v[row]))
        att = torch.zeros(len(where), cfg.q_heads, cfg.head_dim, dtype=torch.float64)
        for row, (b, p) in enumerate(where):
            kk, vv = (torch.stack([t[i] for t in state[li][b][: p + 1]]) for i in (0, 1))
            for h in range(cfg.q_heads):
                kv = h * cfg.kv_heads // cfg.q_heads
                att[row, h] = torch.softmax(kk[:, kv] @ turned[row, h] / cfg.head_dim ** 0.5, -1) @ vv[:, kv]
        x = x + att.reshape(len(where), -1).to(torch.bfloat16).to(x.device) @ w["wo"]
        gu = decode.rmsnorm(x, w["norm2"], cfg.eps) @ w["w_gate_up"]
        inter = gu.shape[1] // 2
        x = x + (torch.nn.functional.silu(gu[:, :inter].float()) * gu[:, inter:].float()).to(torch.bfloat16) @ w["w_down"]
    return x


@pytest.mark.parametrize("fmt", ["int4", "int4-asym", "fp8-tok"])
def test_four_bit_cache_prompt_then_steps(sk, fmt):
    """Prompts of different lengths (one slot empty) in one call, then single tokens, over the 4-bit cache: the
    whole step on this library's operators against plain torch. The same bound as with the bf16 cache, doubled
    for codes that fall on the other side of a border when their input moves by a rounding."""
    from spark_kernels import decode
    from tests import kv4_reference as ref

    cfg = _cfg(sk)
    w = decode.random_weights(cfg, "cuda", seed=15)
    m = decode.QuantizedDecoder(cfg, w, fmt=fmt, batch=3, max_len=40, kv="int4")
    deq = m.dequantized_weights()
    state = [[[] for _ in range(3)] for _ in deq]
    g = torch.Generator(device="cuda").manual_seed(16)
    lens, news = [17, 0, 5], [17, 0, 5]
    for step in range(4):
        off = [0] + torch.tensor(news).cumsum(0).tolist()
        x = torch.randn(off[-1], cfg.hidden, device="cuda", generator=g).to(torch.bfloat16)
        got = m.extend(x, torch.tensor(lens, dtype=torch.int32).cuda(), torch.tensor(off, dtype=torch.int32).cuda()).float()
        want = _reference_step(decode, ref, cfg, deq, state, x, ref.rows_of(lens, off)).float()
        assert ((got - want).norm() / want.norm()).item() < 2 * TOL[fmt], step
        news = [1, 0, 1] if step else [3, 0, 1]
        lens = [a + n for a, n in zip(lens, news)]
    assert sk._C.device_status() == 0


def test_four_bit_cache_graph_replay_equals_eager(sk):
    from spark_kernels import decode

    cfg = _cfg(sk)
    w = decode.random_weights(cfg, "cuda", seed=18)
    eager = decode.QuantizedDecoder(cfg, w, fmt="int4", batch=2, max_len=80, kv="int4")
    graphed = decode.QuantizedDecoder(cfg, w, fmt="int4", batch=2, max_len=80, kv="int4")
    graphed.capture(2)
    g = torch.Generator(device="cuda").manual_seed(19)
    for step in range(70):
        x = torch.randn(2, cfg.hidden, device="cuda", generator=g).to(torch.bfloat16)
        pos = torch.full((2,), step, dtype=torch.int64, device="cuda")
        assert torch.equal(graphed.replay(x, pos), eager.decode(x, pos)), step


def test_cache_formats_are_checked(sk):
    from spark_kernels import decode

    cfg = _cfg(sk)
    w = decode.random_weights(cfg, "cuda", seed=20)
    with pytest.raises(ValueError):
        decode.QuantizedDecoder(cfg, w, kv="int8")
    with pytest.raises(ValueError):
        decode.QuantizedDecoder(cfg, w, batch=1).extend(torch.zeros(1, cfg.hidden, dtype=torch.bfloat16).cuda(), torch.ones(1, dtype=torch.int32).cuda())


def test_four_bit_cache_fewer_sequences_than_slots(sk):
    """A step of the first of three sequences, eager and captured, is the first row's step of a decoder for one."""
    from spark_kernels import decode

    cfg = _cfg(sk)
    w = decode.random_weights(cfg, "cuda", seed=19)
    one = decode.QuantizedDecoder(cfg, w, fmt="fp8-tok", batch=1, max_len=40, kv="int4")
    three = decode.QuantizedDecoder(cfg, w, fmt="fp8-tok", batch=3, max_len=40, kv="int4")
    captured = decode.QuantizedDecoder(cfg, w, fmt="fp8-tok", batch=3, max_len=40, kv="int4")
    captured.capture(1)
    g = torch.Generator(device="cuda").manual_seed(20)
    for t in range(3):
        x, pos = torch.randn(1, cfg.hidden, device="cuda", generator=g).to(torch.bfloat16), torch.tensor([t], device="cuda")
        want = one.decode(x, pos)
        assert torch.equal(three.decode(x, pos), want) and torch.equal(captured.replay(x, pos), want), t
    with pytest.raises(RuntimeError):
        one.extend(torch.randn(2, cfg.hidden, device="cuda").to(torch.bfloat16), torch.ones(2, dtype=torch.int32).cuda())
    assert sk._C.device_status() == 0


@pytest.mark.parametrize("pos", [40, 63, 64, 1000])
def test_four_bit_cache_past_its_length(sk, pos):
    """A position past max_len, inside the sequence's last page and behind it: reported, not written, the other sequence served."""
    from spark_kernels import decode

    cfg = _cfg(sk)
    w = decode.random_weights(cfg, "cuda", seed=21)
    one, two = (decode.QuantizedDecoder(cfg, w, fmt="fp8-tok", batch=n, max_len=40, kv="int4") for n in (1, 2))
    g = torch.Generator(device="cuda").manual_seed(22)
    x = torch.randn(2, cfg.hidden, device="cuda", generator=g).to(torch.bfloat16)
    before = [c.pool.clone() for c in two.cache]
    got = two.decode(x, torch.tensor([pos, 0], device="cuda"))
    assert sk._C.device_status() == 5 and sk._C.device_status() == 0
    assert torch.equal(got[1:], one.decode(x[1:], torch.tensor([0], device="cuda")))
    for c, old, alone in zip(two.cache, before, one.cache):
        assert torch.equal(c.pool[0], old[0]) and torch.equal(c.pool[1], alone.pool[0])
    assert sk._C.device_status() == 0
