"""Attention over the 4-bit cache where a call holds prompts large enough for the kernel that takes 256 rows a block, alone
and beside sequences that the other kernel takes: against 64 bits (tests/kv4_reference.py).

Tolerance: tests/test_kv4.py's covers it. Here keys and values are rounded to fp16 (2^-11 of each): a score is off by at most
2^-11 scale sum|q k|, with |q|, |k| of mean 0.8 at most 2^-11 x 7.3 = 3.6e-3, which moves the output by at most 7.2e-3 vmax;
the values' and the weights' own rounding adds 2 x 2^-11 vmax. Together 8.2e-3 vmax, below the 2.2e-2 vmax there."""

import pytest
import torch

from tests import kv4_reference as ref
from tests.test_kv4 import _attend, _bf16, _check, _filled

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("window", [0, 100])
@pytest.mark.parametrize("d,group", [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128)])
def test_prompts_beside_other_sequences(sk, d, group, window):
    """Two heads a KV head: blocks of 256 rows whole, of 128 and of 2; sequences of one token, of none and of 126 rows between them."""
    g = torch.Generator().manual_seed(d + group + window)
    _check(*_attend(sk, g, [300, 90, 0, 130, 64, 400], [200, 1, 0, 64, 63, 129], 64, 32, 16, d, group, window=window))


@pytest.mark.parametrize("hq,hkv,lens,news", [(16, 16, [260, 413], [257, 300]), (48, 16, [97, 150], [97, 90]), (128, 8, [70, 33], [40, 33]), (40, 8, [300], [220])])
@pytest.mark.parametrize("page", [16, 96])
def test_head_groups_and_pages(sk, hq, hkv, lens, news, page):
    g = torch.Generator().manual_seed(hq + page)
    _check(*_attend(sk, g, lens, news, page, hq, hkv, 128, 64))


def test_rows_before_the_first_token(sk):
    """A sequence that claims more new tokens than it holds: the surplus rows are padding."""
    g = torch.Generator().manual_seed(5)
    got, want, slack = _attend(sk, g, [40, 300], [200, 300], 64, 16, 16, 128, 64)
    assert (got[:160] == 0).all()
    _check(got, want, slack)


def test_magnitudes_and_scale(sk):
    g = torch.Generator().manual_seed(6)
    for mag, scale in ((1e-20, 1e19), (1e20, 1e-21), (1.0, -0.05), (1.0, 0.0), (0.0, 0.1)):
        q = (_bf16(g, 150, 32, 128).float() * mag).to(torch.bfloat16)
        got, want, slack = _attend(sk, g, [150], [150], 16, 32, 16, 128, 64, scale=scale, q=q)
        _check(got, want, slack, f"{mag} {scale}")


def test_sharp_softmax_moves_the_maximum(sk):
    """Scores that grow along the sequence: the running maximum moves in nearly every step."""
    g = torch.Generator().manual_seed(7)
    d, hkv, n = 128, 16, 520
    cache = sk.KV4Cache(9, hkv, d, 64, 64)
    table = torch.randperm(9, generator=g).reshape(1, 9).to(torch.int32)
    x = _bf16(g, n, 2 * hkv * d).float()
    x[:, : hkv * d] = x[:, : hkv * d] * 0.05 + torch.arange(n)[:, None] * 0.02
    lens, off = torch.tensor([n], dtype=torch.int32).cuda(), torch.tensor([0, n], dtype=torch.int32).cuda()
    sk.kv4_append(x.to(torch.bfloat16).cuda(), cache, table.cuda(), lens, None, off)
    q = torch.rand(n, hkv, d, generator=g).to(torch.bfloat16)
    got = sk.kv4_attention(q.cuda(), cache, table.cuda(), lens, off).double().cpu()
    k, v = ref.unpack(cache.pool, d, 64)
    rows = [0, 1, 63, 64, 200, 333, 511, 519]
    for r in rows:
        want, slack = ref.attention(q[r: r + 1], k, v, table.tolist(), [r + 1], None, d ** -0.5, 0)
        # keys of up to 11 and sums of 128 of them: a score of up to 60, rounded by 2^-11 of its terms
        assert ((got[r] - want[0]).abs() <= want[0].abs() * 2 ** -8 + 2 * 60 * 2 ** -11 * slack[0]).all(), r


def test_values_of_very_different_scale(sk):
    g = torch.Generator().manual_seed(8)
    d, hkv, n = 128, 16, 160
    cache = sk.KV4Cache(4, hkv, d, 64, 64)
    table = torch.tensor([[2, 0, 3]], dtype=torch.int32)
    x = _bf16(g, n, 2 * hkv * d).float()
    x[:, hkv * d:] *= torch.exp(6 * torch.randn(n, 1, generator=g))
    lens, off = torch.tensor([n], dtype=torch.int32).cuda(), torch.tensor([0, n], dtype=torch.int32).cuda()
    sk.kv4_append(x.to(torch.bfloat16).cuda(), cache, table.cuda(), lens, None, off)
    q = _bf16(g, n, 2 * hkv, d)
    got = sk.kv4_attention(q.cuda(), cache, table.cuda(), lens, off).double().cpu()
    k, v = ref.unpack(cache.pool, d, 64)
    want, slack = ref.attention(q, k, v, table.tolist(), [n], [0, n], d ** -0.5, 0)
    assert ((got - want).abs() <= want.abs() * 2 ** -8 + (2 ** -10 + 2.2e-2) * slack).all()


def test_nan_reaches_only_its_readers(sk):
    g = torch.Generator().manual_seed(9)
    d, hkv, n = 128, 16, 200
    cache = sk.KV4Cache(9, hkv, d, 64, 64)
    table = torch.randperm(9, generator=g)[:8].reshape(2, 4).to(torch.int32).cuda()
    x = _bf16(g, 2 * n, 2 * hkv * d)
    x[70, hkv * d + 3] = float("nan")       # V of head 0, token 70 of sequence 0, first group
    x[90, 5 * d + 100] = float("inf")       # K of head 5, token 90 of sequence 0
    lens, off = torch.tensor([n, n], dtype=torch.int32).cuda(), torch.tensor([0, n, 2 * n], dtype=torch.int32).cuda()
    sk.kv4_append(x.cuda(), cache, table, lens, None, off)
    q = _bf16(g, 2 * n, 2 * hkv, d).cuda()
    q[n + 7, 3, 5] = float("nan")
    for window in (0, 10):
        out = torch.isnan(sk.kv4_attention(q, cache, table, lens, off, window=window)).cpu()
        want = torch.zeros_like(out)
        want[70: n if not window else 80, 0:2, :64] = True
        want[90: n if not window else 100, 10:12] = True
        want[n + 7, 3] = True
        assert torch.equal(out, want), window


def test_bad_pages_rest_and_given_out(sk):
    g = torch.Generator().manual_seed(10)
    d, hkv = 128, 16
    cache, table = _filled(sk, g, [300, 300], 64, hkv, d, 64)
    q = _bf16(g, 400, 32, d).cuda()
    lens, off = torch.tensor([300, 300], dtype=torch.int32).cuda(), torch.tensor([0, 200, 390], dtype=torch.int32).cuda()
    good = sk.kv4_attention(q, cache, table.cuda(), lens, off)
    assert sk._C.device_status() == 0 and (good[390:] == 0).all()
    out = torch.full_like(q, 7.0)
    sk.kv4_attention(q, cache, table.cuda(), lens, off, out=out)
    assert torch.equal(out[:390], good[:390]) and (out[390:] == 7).all()
    for bad in (-1, cache.pages, 1 << 30):
        broken = table.clone()
        broken[0, 1] = bad
        got = sk.kv4_attention(q, cache, broken.cuda(), lens, off)
        assert sk._C.device_status() == 5
        assert torch.equal(got[200:390], good[200:390]) and torch.isfinite(got).all()
    got = sk.kv4_attention(q, cache, table.cuda(), torch.tensor([1 << 30, 300], dtype=torch.int32).cuda(), off)
    assert sk._C.device_status() == 5 and torch.equal(got[200:390], good[200:390])


def test_same_bits_captured_and_with_other_streams(sk):
    g = torch.Generator().manual_seed(11)
    cache, table = _filled(sk, g, [900, 40], 64, 16, 128, 64)
    t, lens, off = table.cuda(), torch.tensor([900, 40], dtype=torch.int32).cuda(), torch.tensor([0, 600, 601], dtype=torch.int32).cuda()
    q = _bf16(g, 601, 32, 128).cuda()
    want = sk.kv4_attention(q, cache, t, lens, off)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = sk.kv4_attention(q, cache, t, lens, off)
    sides = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for _ in range(3):
        graph.replay()
        for s in sides:
            with torch.cuda.stream(s):
                outs.append(sk.kv4_attention(q, cache, t, lens, off))
    torch.cuda.synchronize()
    assert torch.equal(got, want) and all(torch.equal(o, want) for o in outs)
    # lengths read on the device at replay: the prompt becomes a single token, and nothing is left of it; the other sequence now
    # reads tokens that were never written, NaN among them, hence the comparison of bits
    lens.copy_(torch.tensor([17, 900], dtype=torch.int32)), off.copy_(torch.tensor([0, 1, 601], dtype=torch.int32))
    graph.replay()
    assert torch.equal(got.view(torch.int16), sk.kv4_attention(q, cache, t, lens, off).view(torch.int16))


@pytest.mark.parametrize("size", [2.0 ** 125, 2.0 ** 126, 2.0 ** 127, 2.0 ** -100, 2.0 ** -126])
def test_values_at_the_ends_of_the_range(sk, size):
    """Values between one and one and a half times `size` (of the least, groups have no scale left and are their minimum) in a
    prompt: as near to 64 bits as others, relative to the values."""
    g = torch.Generator().manual_seed(12)
    d, hkv, n = 128, 16, 150
    cache = sk.KV4Cache(3, hkv, d, 64, 64)
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32)
    x = _bf16(g, n, 2 * hkv * d)
    x[:, hkv * d:] = ((1 + 0.5 * torch.rand(n, hkv * d, generator=g)).double() * size).to(torch.bfloat16)
    lens, off = torch.tensor([n], dtype=torch.int32).cuda(), torch.tensor([0, n], dtype=torch.int32).cuda()
    sk.kv4_append(x.cuda(), cache, table.cuda(), lens, None, off)
    q = _bf16(g, n, 2 * hkv, d)
    got = sk.kv4_attention(q.cuda(), cache, table.cuda(), lens, off).double().cpu() / size
    k, v = ref.unpack(cache.pool, d, 64)
    want, slack = ref.attention(q, k, v / size, table.tolist(), [n], [0, n], d ** -0.5, 0)
    assert ((got - want).abs() <= want * 2 ** -8 + (2 ** -10 + 2.2e-2) * slack).all()
