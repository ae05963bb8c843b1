"""Attention over the 4-bit cache at the ends of the numbers' range, against 64 bits (tests/kv4_reference.py), in the kernel
for few rows and in the one for prompts. Tolerances: tests/test_kv4.py's (which covers the prompts', tests/test_kv4_prompts.py),
whose slack is a channel's own largest value, so that quiet channels are not measured against loud ones."""

import pytest
import torch

from tests import kv4_reference as ref
from tests.test_kv4 import _attend, _bf16, _check

pytestmark = pytest.mark.gpu

# lens, new tokens, query heads, KV heads: two tokens of a decode step, and 32 blocks of a prompt
FEW, PROMPT = ([200, 40], None, 4, 2), ([150], [150], 32, 16)


@pytest.mark.parametrize("lens,news,hq,hkv", [FEW, PROMPT])
@pytest.mark.parametrize("power", [-133, -126, -120, -113, 100, 120])
def test_queries_at_the_ends_of_the_range(sk, lens, news, hq, hkv, power):
    """Queries of up to 127 x 2^power (at -133: below the normal numbers) with a scale that makes the scores ordinary. The scores'
    error bound scales with |scale q|, whose mean is 0.8 d^-1/2 here as there."""
    g = torch.Generator().manual_seed(power + 200)
    rows = len(lens) if news is None else sum(news)
    n = (40 * torch.randn(rows, hq, 128, generator=g)).round().clamp(-127, 127)
    q = (n.double() * 2.0 ** power).to(torch.bfloat16)
    assert torch.equal(q.double(), n.double() * 2.0 ** power)
    got, want, slack = _attend(sk, g, lens, news, 16, hq, hkv, 128, 64, scale=2.0 ** -power / 40 * 128 ** -0.5, q=q)
    _check(got, want, slack, f"2^{power}")


def _cache(sk, g, n, hkv, d, group, spoil, page=64):
    """One sequence of n tokens appended to a cache; spoil(x [n, 2, hkv, d]) changes its keys and values before."""
    pages = -(-n // page)
    cache = sk.KV4Cache(pages + 2, hkv, d, page, group)
    table = torch.randperm(pages + 2, generator=g)[:pages].reshape(1, pages).to(torch.int32)
    x = torch.randn(n, 2, hkv, d, generator=g)
    spoil(x)
    off = torch.tensor([0, n], dtype=torch.int32).cuda()
    sk.kv4_append(x.to(torch.bfloat16).reshape(n, -1).cuda(), cache, table.cuda(), torch.tensor([n], dtype=torch.int32).cuda(), None, off)
    return cache, table


def _attend_last(sk, cache, table, n, q, scale, rows):
    """q [new tokens, heads, d], the sequence's last ones -> (got, want, slack) of the named rows."""
    news = q.shape[0]
    off = None if news == 1 else torch.tensor([0, news], dtype=torch.int32).cuda()
    got = sk.kv4_attention(q.cuda(), cache, table.cuda(), torch.tensor([n], dtype=torch.int32).cuda(), off, scale=scale)
    k, v = ref.unpack(cache.pool, cache.head_dim, cache.group)
    parts = [ref.attention(q[r: r + 1], k, v, table.tolist(), [n - news + r + 1], None, scale, 0) for r in rows]
    return got[rows], torch.cat([p[0] for p in parts]), torch.cat([p[1] for p in parts])


def _check_groups(got, want, slack, group, what, held=0.0):
    """_check of every group by itself; held: what an output may be off by besides."""
    for at in range(0, got.shape[-1], group):
        g, w, s = (t[..., at: at + group] for t in (got, want, slack))
        if held == 0.0:
            _check(g, w, s, f"{what}, channels {at}..")
            continue
        off = (g.double().cpu() - w).abs()
        assert torch.isfinite(g).all() and (off <= w.abs() * 2 ** -8 + (2 ** -11 + 2.2e-2) * s + held).all(), f"{what}, channels {at}.."
        assert off.norm() <= 1.5 * 2 ** -8 * w.norm() + held * w.numel() ** 0.5, f"{what}, channels {at}.."


@pytest.mark.parametrize("n,news,hq,hkv", [(200, 1, 4, 2), (60000, 1, 4, 2), (400, 150, 32, 16)])
@pytest.mark.parametrize("which", ["keys", "values"])
def test_scales_below_zero(sk, n, news, hq, hkv, which):
    """A pool of the caller's whose scales are negative or -0 in a third of the tiles each: c * scale + minimum all the same. The
    keys are then up to three times as large: a quarter of the usual scale keeps the scores' error below its bound."""
    g = torch.Generator().manual_seed(31)
    d, group = 128, 64
    cache, table = _cache(sk, g, n, hkv, d, group, lambda x: None)
    at = 16 * d + (64 * (d // group) if which == "values" else 0)
    words = cache.pool[..., at: at + 64 * (d // group)].contiguous().view(torch.bfloat16)  # ..., minimum, scale, ...
    s = words[..., 1::2]
    kind = torch.randint(0, 3, (*s.shape[:3], 1), generator=g).cuda()
    words[..., 1::2] = torch.where(kind == 0, s, torch.where(kind == 1, -s, torch.full_like(s, -0.0)))
    cache.pool[..., at: at + 64 * (d // group)] = words.view(torch.uint8)
    got, want, slack = _attend_last(sk, cache, table, n, _bf16(g, news, hq, d), 0.25 * d ** -0.5, list(range(0, news, 7)))
    _check(got, want, slack, which)


def _opposed(x, at):
    """Token `at` gets keys that every query of positive channels scores far below the others: its weight is nothing."""
    x[at, 0] = -3


@pytest.mark.parametrize("n", [150, 30000])
@pytest.mark.parametrize("power", [8, 12, 16, 20, 40])
@pytest.mark.parametrize("hq,hkv,d,group", [(4, 1, 128, 64), (4, 1, 128, 32), (8, 1, 128, 32), (16, 1, 64, 32), (3, 1, 64, 32), (2, 1, 64, 64), (16, 1, 128, 128)])
def test_quiet_values_beside_loud_ones(sk, hq, hkv, d, group, power, n):
    """Values of the first 32 channels (all of them where they are one group) 2^power louder: of the whole sequence, of one token with
    an ordinary weight, of one token with next to none. Every group of channels is as near to 64 bits as it would be alone."""
    def every(x):
        x[:, 1, :, :32] *= 2.0 ** power

    def one(x):
        x[3, 1, :, :32] *= 2.0 ** power

    def weightless(x):
        x[3, 1, :, :32] *= 2.0 ** power
        _opposed(x, 3)

    g = torch.Generator().manual_seed(power + n)
    for spoil in (every, one, weightless):
        cache, table = _cache(sk, g, n, hkv, d, group, spoil)
        q = _bf16(g, 1, hq, d).abs()
        got, want, slack = _attend_last(sk, cache, table, n, q, d ** -0.5, [0])
        _check_groups(got, want, slack, group, spoil.__name__)


@pytest.mark.parametrize("power", [12, 18, 30])
@pytest.mark.parametrize("hq,d,group", [(64, 128, 64), (160, 64, 32), (320, 128, 64)])
def test_quiet_values_beside_loud_ones_in_long_ranges(sk, hq, d, group, power):
    """The same where a warp reads some 250 tokens of a head on its own: loud groups, and every 50th token loud and nearly without weight."""
    n, hkv = 16000, 32

    def every(x):
        x[:, 1, :, :32] *= 2.0 ** power

    def weightless(x):
        x[::50, 1, :, :32] *= 2.0 ** power
        _opposed(x, slice(None, None, 50))

    g = torch.Generator().manual_seed(power)
    for spoil in (every, weightless):
        cache, table = _cache(sk, g, n, hkv, d, group, spoil)
        q = _bf16(g, 1, hq, d).abs()
        got = sk.kv4_attention(q.cuda(), cache, table.cuda(), torch.tensor([n], dtype=torch.int32).cuda())[:, : hq // hkv]
        k, v = ref.unpack(cache.pool[:, :1], d, group)
        want, slack = ref.attention(q[:, : hq // hkv], k, v, table.tolist(), [n], None, d ** -0.5, 0)
        _check_groups(got, want, slack, group, spoil.__name__)


@pytest.mark.parametrize("n", [150, 4000])
@pytest.mark.parametrize("power", [8, 12, 16, 20, 28])
@pytest.mark.parametrize("d,group", [(128, 64), (64, 32), (128, 128), (128, 32), (64, 64)])
def test_quiet_values_beside_loud_ones_in_prompts(sk, d, group, power, n):
    """In prompts a value is c s' + m' in fp16, s' and m' being the group's times 2^(14 - e), 2^e the power above the largest |m| + 15 s of its
    16 tokens. Where s' and m' are below fp16's normal numbers each is off by up to 2^-25, and so is the result: 17 x 2^-25 x 2^(e - 14) of
    the value. |m| is at most the largest |v|, 15 s at most twice that and a rounding: 2^e is at most 2 x 3.03 of it and the
    value off by at most 2^-32 of the largest value."""
    def every(x):
        x[:, 1, :, :32] *= 2.0 ** power

    def one(x):
        x[3, 1, :, :32] *= 2.0 ** power

    def weightless(x):
        x[3, 1, :, :32] *= 2.0 ** power
        _opposed(x, 3)

    g = torch.Generator().manual_seed(power + n)
    for spoil in (every, one, weightless):
        cache, table = _cache(sk, g, n, 16, d, group, spoil)
        q = _bf16(g, 150, 32, d).abs()
        got, want, slack = _attend_last(sk, cache, table, n, q, d ** -0.5, [20, 149])
        _check_groups(got, want, slack, group, spoil.__name__, held=2.0 ** -32 * slack.amax().item())


@pytest.mark.parametrize("n", [20, 64, 60000])
def test_values_that_are_no_numbers_under_weights_that_vanish(sk, n):
    """A value that is a NaN spoils the rows that see it whatever its weight: 0 x NaN is no number. The first two lengths are read in
    steps with tokens out of sight; the last is cut over all CTAs, most of them without the token."""
    g = torch.Generator().manual_seed(33)

    def spoil(x):
        x[5, 0] = -30  # scores below -300: a weight that fp32 does not hold
        x[5, 1, 0, 3] = float("nan")

    cache, table = _cache(sk, g, n, 2, 128, 64, spoil)
    q = 1 + _bf16(g, 1, 4, 128).abs()
    out = torch.isnan(sk.kv4_attention(q.cuda(), cache, table.cuda(), torch.tensor([n], dtype=torch.int32).cuda()).cpu())
    want = torch.zeros_like(out)
    want[:, :2, :64] = True
    assert torch.equal(out, want)


@pytest.mark.parametrize("first", [1.0, 0.0])
def test_many_small_weights_beside_a_large_one_in_prompts(sk, first):
    """A key at 2^25.1 times the weight of each of 2^18 others, which together have 1 % of the sum. Its value is 1 or 0, theirs 1: the
    output is 1 or that percent. Keys and values are exact in fp16 here; the large weight is 2^4, the others 2^-21.1 in steps of 2^-24:
    off by up to 2^-25, 2^-3.8 of them. The values' products are 2^13 times that, summed in fp32. A sum of 2^17, which the large one
    makes, ends at 2^-6 and may drop each of the others, 2^-8.1, whole; without it the sum ends below 2^10, its last bit is 2^-14
    and may be cut off each, 2^-5.8 of it."""
    d, hkv, page, n = 128, 16, 1024, 1 << 18
    cache = sk.KV4Cache(4, hkv, d, page, 64)
    x = torch.ones(2 * page, 2, hkv, d)
    x[:, 0] = 0
    x[0, 0] = 1.5390625  # its score is 128 x that x 128^-1/2 = 25.12 ln 2
    x[0, 1] = first
    off, lens = torch.tensor([0, 2 * page], dtype=torch.int32).cuda(), torch.tensor([2 * page], dtype=torch.int32).cuda()
    sk.kv4_append(x.reshape(2 * page, -1).to(torch.bfloat16).cuda(), cache, torch.tensor([[3, 1]], dtype=torch.int32).cuda(), lens, None, off)
    table = torch.tensor([[3] + (n // page - 1) * [1]], dtype=torch.int32).cuda()  # pages may be shared for reading
    q = torch.ones(150, 2 * hkv, d, dtype=torch.bfloat16).cuda()
    got = sk.kv4_attention(q, cache, table, torch.tensor([n], dtype=torch.int32).cuda(), torch.tensor([0, 150], dtype=torch.int32).cuda()).double().cpu()
    small = (n - 150 + torch.arange(150, dtype=torch.float64)) * 2.718281828459045 ** (-1.5390625 * 128 ** 0.5)
    want = ((first + small) / (1 + small))[:, None, None]
    tol = 2 ** -9 + 2 ** -11 + small / (1 + small) if first else want.flatten() * (2 ** -8 + 2 ** -3.8 + 2 ** -5.8)
    assert ((got - want).abs() <= tol[:, None, None]).all(), got.aminmax()


@pytest.mark.parametrize("n,news,hq,hkv,power", [(200, 1, 4, 2, p) for p in (12, 16, 20, 24, 28)] + [(300, 1, 20, 2, 28)] + [(200, 150, 32, 16, p) for p in (12, 16, 20)])
def test_quiet_queries_of_loud_keys(sk, n, news, hq, hkv, power):
    """The second group's queries 2^power quieter than the first's and its keys as much louder: both have their part in the scores. In prompts
    a key is held to 2^-32 of the largest of its 16 tokens' (see the values below), which times 2^20 and a sum of |q| is nothing."""
    def spoil(x):
        x[:, 0, :, 64:] *= 2.0 ** power

    g = torch.Generator().manual_seed(power)
    cache, table = _cache(sk, g, n, hkv, 128, 64, spoil)
    q = torch.randn(news, hq, 128, generator=g)
    q[..., 64:] *= 2.0 ** -power
    q = q.to(torch.bfloat16)
    _check(*_attend_last(sk, cache, table, n, q, 128 ** -0.5, list(range(0, news, 31))), f"2^{power}")


@pytest.mark.parametrize("lens,news,hq,hkv", [FEW, PROMPT])
@pytest.mark.parametrize("scale", [2.5e38, 3e38, -3e38])
def test_scales_of_the_scores_at_the_end_of_the_range(sk, lens, news, hq, hkv, scale):
    """As large as the entry takes, with queries below the normal numbers: n 2^-133 x 3e38 is n / 36, and n is some three in size."""
    g = torch.Generator().manual_seed(41)
    rows = len(lens) if news is None else sum(news)
    q = ((3 * torch.randn(rows, hq, 128, generator=g)).round().double() * 2.0 ** -133).to(torch.bfloat16)
    got, want, slack = _attend(sk, g, lens, news, 16, hq, hkv, 128, 64, scale=scale, q=q)
    _check(got, want, slack, f"{scale}")



@pytest.mark.parametrize("n,news,hq,hkv", [(200, 1, 4, 2), (300, 1, 20, 2), (200, 150, 32, 16)])
@pytest.mark.parametrize("power", [60, 100, 112])
def test_huge_keys_of_tiny_queries(sk, n, news, hq, hkv, power):
    """Keys 2^power and queries 2^-power times the usual: ordinary scores, through sums that stay inside fp32."""
    def spoil(x):
        x[:, 0] *= 2.0 ** power

    g = torch.Generator().manual_seed(power)
    cache, table = _cache(sk, g, n, hkv, 128, 64, spoil)
    q = (torch.randn(news, hq, 128, generator=g) * 2.0 ** -power).to(torch.bfloat16)
    _check(*_attend_last(sk, cache, table, n, q, 128 ** -0.5, list(range(0, news, 31))), f"2^{power}")


@pytest.mark.parametrize("n,news,hq,hkv", [(3000, 1, 4, 2), (3000, 1, 20, 2), (9000, 3, 8, 1), (3000, 150, 32, 16)])
@pytest.mark.parametrize("scale", [1e4, 1e6, 1e7, 1e9, 1e20, -1e12, 1e36])
def test_scores_so_large_that_one_token_has_all_the_weight(sk, n, news, hq, hkv, scale):
    """Where a row's largest q . k stands out by 2, more than the sums' errors (|q . k| is some 50, a sum of 128 |q k| some 80, off by
    at most 2^-11 of that), its output is that token's value: rounded to bf16, behind a weight times scale and a value in fp16 (2^-11
    each of c s + 8 s + m or so: 2^-9 of the largest value). Where none does it is a mean of values."""
    g = torch.Generator().manual_seed(51)
    d = 128
    cache, table = _cache(sk, g, n, hkv, d, 64, lambda x: None)
    q = _bf16(g, news, hq, d)
    off = None if news == 1 else torch.tensor([0, news], dtype=torch.int32).cuda()
    got = sk.kv4_attention(q.cuda(), cache, table.cuda(), torch.tensor([n], dtype=torch.int32).cuda(), off, scale=scale).double().cpu()
    k, v = (t[table[0].long()].flatten(0, 1)[:n] for t in ref.unpack(cache.pool, d, 64))
    assert torch.isfinite(got).all()
    sure = 0
    for r in range(0, news, 17):
        for h in range(hq):
            s = k[: n - news + r + 1, h * hkv // hq] @ q[r, h].double() * (1 if scale > 0 else -1)
            best = s.topk(2)
            vv = v[: len(s), h * hkv // hq]
            assert (got[r, h].abs() <= vv.abs().amax(0) * (1 + 2 ** -7)).all()
            if best.values[0] - best.values[1] > 2:
                sure += 1
                want = vv[best.indices[0]]
                assert ((got[r, h] - want).abs() <= want.abs() * 2 ** -8 + 2 ** -9 * vv.abs().amax(0)).all(), (r, h)
    assert sure > 0
