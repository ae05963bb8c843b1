"""The 4-bit paged KV cache: append, read and attention against plain forms in 64 bits (tests/kv4_reference.py).

Tolerances. A bf16 output is off by half a step of its own, 2^-8 of it. `kv4_read` is one rounding of exact values, the
codes and words of bf16 inputs are exact, so values are compared for equality with the rounded 64-bit ones.
Attention: the weights are rounded to fp16 (2^-11 each, against values of at most vmax: 2^-11 vmax in the output). Scores:
a group's products q'(1024 + c) are exact in fp32 (11 x 11 bits) and summed by at most group / 16 + 1 <= 9 steps, each off by
at most 2^-22 of a partial sum of at most 1039 sum|q'|: 9 x 1039 x 2^-22 = 2.3e-3 of scale s sum|q|. The inputs below have
|q| of mean 0.8, s of at most 0.5 and scale d^-1/2, which makes scale s sum|q| at most 0.5 x 0.8 x 128^1/2 = 4.6 and the
score off by at most 1.1e-2; signs alternate, and a fiftieth of that is the root mean square. A score error e moves the
output by at most 2 e vmax. Per element: 2^-8 |out| + (2^-11 + 2 x 1.1e-2) vmax. Over a whole output (2-norm) the rounding
steps are independent: half a step of bf16 alone is at most 2^-8 of the norm, and 2^-8 x 1.5 is the bound there."""

import pytest
import torch

from tests import kv4_reference as ref

pytestmark = pytest.mark.gpu

SHAPES = [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128)]


def _bf16(g, *shape):
    return torch.randn(shape, generator=g).to(torch.bfloat16)


def _table(g, seqs, width, pages):
    return torch.randperm(pages, generator=g)[: seqs * width].reshape(seqs, width).to(torch.int32)


def _filled(sk, g, lens, page, heads, d, group, spare=2):
    """A cache whose sequences hold random tokens, written by kv4_append, with every byte that was never written 0xff
    (a NaN wherever it is read as a scale)."""
    width = max(1, -(-max(lens) // page))
    pages = len(lens) * width + spare
    table = _table(g, len(lens), width, pages)
    cache = sk.KV4Cache(pages, heads, d, page, group)
    cache.pool.fill_(255)
    rows = sum(lens)
    off = torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32)
    if rows:
        sk.kv4_append(_bf16(g, rows, 2 * heads * d).cuda(), cache, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), None, off.cuda())
    return cache, table


def _check(got, want, slack, what=""):
    got = got.double().cpu()
    assert torch.isfinite(got).all(), what
    bound = want.abs() * 2 ** -8 + (2 ** -11 + 2.2e-2) * slack + 1e-30
    bad = (got - want).abs() > bound
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} out of bounds"
    if want.norm() > 0:
        assert ((got - want).norm() / want.norm()).item() < 1.5 * 2 ** -8, what


def _attend(sk, g, lens, news, page, hq, hkv, d, group, window=0, scale=None, q=None):
    cache, table = _filled(sk, g, lens, page, hkv, d, group)
    offs = None if news is None else [0] + torch.tensor(news).cumsum(0).tolist()
    rows = len(lens) if news is None else offs[-1]
    q = _bf16(g, rows, hq, d) if q is None else q
    got = sk.kv4_attention(q.cuda(), cache, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(),
                           None if offs is None else torch.tensor(offs, dtype=torch.int32).cuda(), scale=scale, window=window)
    k, v = ref.unpack(cache.pool, d, group)
    want, slack = ref.attention(q, k, v, table.tolist(), lens, offs, d ** -0.5 if scale is None else scale, window)
    assert sk._C.device_status() == 0
    return got, want, slack


@pytest.mark.parametrize("d,group", SHAPES)
@pytest.mark.parametrize("rot", ["all", "half", "some", "none"])
def test_append_and_read(sk, d, group, rot):
    g = torch.Generator().manual_seed(d + group)
    hq, hkv, page = 5, 3, 32
    lens, news = [70, 0, 33, 1, 5], [13, 0, 33, 1, 4]
    off = torch.tensor([0] + torch.tensor(news).cumsum(0).tolist(), dtype=torch.int32)
    rows = int(off[-1])
    table = _table(g, 5, 3, 17)
    n_rot = {"all": d, "half": d // 2, "some": 24, "none": 0}[rot]
    cs = None if n_rot == 0 else torch.cat([f(torch.arange(100)[:, None] * 0.37 ** torch.arange(n_rot // 2)) for f in (torch.cos, torch.sin)], 1).float()
    qkv = _bf16(g, rows, (hq + 2 * hkv) * d)
    qkv[:, hq * d: (hq + hkv) * d: 11] *= 8
    cache = sk.KV4Cache(17, hkv, d, page, group)
    q = sk.kv4_append(qkv.cuda(), cache, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), None if cs is None else cs.cuda(), off.cuda())
    where = ref.rows_of(lens, off.tolist())
    slots = torch.tensor([int(table[b, p // page]) * page + p % page for b, p in where])
    k, v = sk.kv4_read(cache, slots.cuda())
    x = qkv.double().reshape(rows, -1, d)
    if cs is not None:
        pos = torch.tensor([p for _, p in where])
        x = torch.cat([ref.rotate(x[:, : hq + hkv], cs[pos]), x[:, hq + hkv:]], 1)
    assert ((q.cpu().double() - x[:, :hq]).abs() <= x[:, :hq].abs() * 2 ** -8 + 2.0 ** -22 * x.abs().amax()).all()
    want_v, _, _ = ref.quantize(x[:, hq + hkv:], group)
    assert torch.equal(v.cpu(), want_v.to(torch.bfloat16))
    # keys are rotated in fp32: a code next to a border may fall on its other side, so a value is held to what a code may be off by
    y = x[:, hq: hq + hkv]
    want_k, s, m = ref.quantize(y, group)
    near = ((((y - m) / s) % 1) - 0.5).abs() < 1e-4
    same = k.cpu() == want_k.to(torch.bfloat16)
    assert (same | near).float().mean() > 0.999 and same.float().mean() > 0.995
    assert ((k.cpu().double() - want_k).abs() <= want_k.abs() * 2 ** -8 + s * (1 + 2 ** -7) + 15 * s * 2 ** -7).all()
    assert sk._C.device_status() == 0
    # the bytes themselves, by their documented places
    kk, vv = ref.unpack(cache.pool, d, group)
    assert torch.equal(vv.reshape(-1, hkv, d)[slots].to(torch.bfloat16), v.cpu()) and torch.equal(kk.reshape(-1, hkv, d)[slots].to(torch.bfloat16), k.cpu())


@pytest.mark.parametrize("d,group", [(64, 64), (128, 32), (128, 128)])
def test_append_odd_groups(sk, d, group):
    """Groups of one value, of a huge offset, of extreme magnitudes, with infinities and NaN; what is not appended stays."""
    g = torch.Generator().manual_seed(3)
    x = _bf16(g, 9, 2 * d).float()
    x[0] = 0
    x[1] = -3.171875
    x[2] = 1000 + x[2]
    x[3] *= 1e-39
    x[4] *= 1e37
    x[5, 3], x[5, d + 5] = float("inf"), float("-inf")
    x[6, 7] = float("nan")
    x[7, 0], x[7, 1] = 3.38e38, -3.38e38  # a range past fp32
    x[8] *= 2.0 ** -120
    x = x.to(torch.bfloat16)
    cache = sk.KV4Cache(2, 1, d, 16, group)
    cache.pool.fill_(0x5a)
    before = cache.pool.clone()
    off = torch.tensor([0, 9], dtype=torch.int32).cuda()
    sk.kv4_append(x.cuda(), cache, torch.tensor([[1]], dtype=torch.int32).cuda(), torch.tensor([9], dtype=torch.int32).cuda(), None, off)
    k, v = sk.kv4_read(cache, torch.arange(16, 25).cuda())
    got = torch.cat([k[:, 0], v[:, 0]], 1).cpu()
    gr = x.double().unflatten(-1, (-1, group))
    m = gr.amin(-1, keepdim=True)
    bad = (~torch.isfinite(gr)).any(-1, keepdim=True) | ~torch.isfinite((gr.amax(-1, keepdim=True) - m).float())
    want = torch.where(bad, torch.full((), float("nan"), dtype=torch.float64), ref.quantize(x.double(), group)[0].unflatten(-1, (-1, group))).flatten(-2).to(torch.bfloat16)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got[~torch.isnan(want)], want[~torch.isnan(want)])
    assert torch.equal(cache.pool[0], before[0])          # the other page
    assert torch.equal(sk.kv4_read(cache, torch.arange(25, 32).cuda())[0].isnan(), sk.kv4_read(sk.KV4Cache.from_pool(before, d, group), torch.arange(25, 32).cuda())[0].isnan())


def test_append_strides_padding_and_rest(sk):
    """Strided rows; rows behind the last sequence; empty slots; a q_out of the caller's."""
    g = torch.Generator().manual_seed(4)
    d, hq, hkv = 128, 4, 2
    wide = _bf16(g, 6, (hq + 2 * hkv) * d + 64).cuda()
    qkv = wide[:, 64:]
    table = torch.arange(4, dtype=torch.int32).reshape(4, 1).cuda()
    lens = torch.tensor([3, 0, 2, 1], dtype=torch.int32).cuda()
    off = torch.tensor([0, 2, 2, 3, 4], dtype=torch.int32).cuda()
    a, b = sk.KV4Cache(4, hkv, d, 16, 64), sk.KV4Cache(4, hkv, d, 16, 64)
    cs = sk.kv4.rotation_table(8, d).cuda()
    out = torch.full((6, hq, d), 7.0, dtype=torch.bfloat16, device="cuda")
    assert sk.kv4_append(qkv, a, table, lens, cs, off, q_out=out) is out
    fresh = sk.kv4_append(qkv.contiguous(), b, table, lens, cs, off)
    assert torch.equal(a.pool, b.pool) and torch.equal(out[:4], fresh[:4])
    assert (out[4:] == 7).all() and (fresh[4:] == 0).all()
    # one row per sequence: the slot of length 0 is padding
    c = sk.KV4Cache(4, hkv, d, 16, 64)
    one = sk.kv4_append(qkv[:4], c, table, lens, cs)
    assert (one[1] == 0).all() and (c.pool[1] == 0).all() and (c.pool[0] != 0).any()


@pytest.mark.parametrize("d,group", SHAPES)
@pytest.mark.parametrize("hq,hkv", [(8, 2), (3, 3), (16, 1), (7, 1), (40, 2)])
def test_decode_attention(sk, d, group, hq, hkv):
    g = torch.Generator().manual_seed(hq * d + group)
    lens = [1, 0, 2, 15, 16, 17, 63, 64, 65, 130, 700]
    _check(*_attend(sk, g, lens, None, 32, hq, hkv, d, group), f"d={d} group={group} heads={hq}/{hkv}")


@pytest.mark.parametrize("page", [16, 48, 64, 256])
@pytest.mark.parametrize("window", [0, 1, 16, 100])
def test_pages_and_windows(sk, page, window):
    g = torch.Generator().manual_seed(page + window)
    _check(*_attend(sk, g, [300, 1, 99, 0, 17], None, page, 4, 2, 128, 64, window=window), f"page={page} window={window}")


@pytest.mark.parametrize("window", [0, 7, 40])
@pytest.mark.parametrize("hq,hkv,d,group", [(8, 2, 128, 64), (4, 4, 64, 32), (5, 1, 128, 128), (16, 1, 64, 64)])
def test_several_tokens_a_sequence(sk, hq, hkv, d, group, window):
    """Chunks of different lengths on caches of different lengths, a whole prompt, an empty sequence, and a sequence
    whose rows reach back before its first token (padding)."""
    g = torch.Generator().manual_seed(hq + window)
    lens, news = [90, 33, 0, 200, 5, 2], [3, 33, 0, 37, 1, 4]
    _check(*_attend(sk, g, lens, news, 32, hq, hkv, d, group, window=window), f"window={window}")


@pytest.mark.parametrize("lens,news", [([700], [600]), ([260, 513], [257, 128]), ([129], [129])])
@pytest.mark.parametrize("hq,hkv,d,group", [(4, 1, 128, 64), (2, 2, 64, 64), (3, 1, 128, 32), (4, 1, 64, 32), (2, 1, 128, 128)])
def test_prompts(sk, lens, news, hq, hkv, d, group):
    g = torch.Generator().manual_seed(sum(lens) + hq)
    for window in (0, 150):
        _check(*_attend(sk, g, lens, news, 64, hq, hkv, d, group, window=window), f"{lens} {news} window={window}")


def test_magnitudes_and_scale(sk):
    """Queries far from 1, a scale of the caller's (negative too), sharp softmaxes."""
    g = torch.Generator().manual_seed(12)
    for mag, scale in ((1e-20, 1e19), (1e20, 1e-21), (1.0, -0.05), (1.0, 0.0)):
        q = (_bf16(g, 3, 4, 128).float() * mag).to(torch.bfloat16)
        got, want, slack = _attend(sk, g, [200, 40, 3], None, 16, 4, 2, 128, 64, scale=scale, q=q)
        _check(got, want, slack, f"{mag} {scale}")


def test_values_of_very_different_scale(sk):
    """Values whose groups and tokens differ in magnitude by many orders: the softmax weights carry the scales."""
    g = torch.Generator().manual_seed(13)
    d, lens = 128, [150]
    cache = sk.KV4Cache(4, 1, d, 64, 64)
    table = torch.tensor([[2, 0, 3]], dtype=torch.int32).cuda()
    x = _bf16(g, 150, 2 * d).float()
    x[:, d: d + 64] *= torch.exp(8 * torch.randn(150, 1, generator=g))
    x[:, d + 64:] *= 1e-6
    off = torch.tensor([0, 150], dtype=torch.int32).cuda()
    lt = torch.tensor(lens, dtype=torch.int32).cuda()
    sk.kv4_append(x.to(torch.bfloat16).cuda(), cache, table, lt, None, off)
    q = _bf16(g, 1, 4, d)
    got = sk.kv4_attention(q.cuda(), cache, table, lt).cpu().double()
    k, v = ref.unpack(cache.pool, d, 64)
    want, slack = ref.attention(q, k, v, table.tolist(), lens, None, d ** -0.5, 0)
    # the weights' range: 2^-24 of the largest weight times scale of the tile's tokens is what rounding to fp16 leaves of the
    # other group's, here below the group's own slack only for the loud one; the quiet one is held to the loud one's rounding
    loud = slack.amax()
    assert ((got - want).abs() <= want.abs() * 2 ** -8 + (2 ** -11 + 2.2e-2) * slack + 2.0 ** -24 * loud).all()


def test_strided_queries_given_out_and_rest(sk):
    g = torch.Generator().manual_seed(14)
    d, hq = 128, 4
    cache, table = _filled(sk, g, [40, 20], 16, 2, d, 64)
    wide = _bf16(g, 5, (hq + 3) * d).cuda()
    q = wide[:, d: (hq + 1) * d].unflatten(1, (hq, d))
    lens, off = torch.tensor([40, 20], dtype=torch.int32).cuda(), torch.tensor([0, 1, 3], dtype=torch.int32).cuda()
    plain = sk.kv4_attention(q.contiguous(), cache, table.cuda(), lens, off)
    out = torch.full((5, hq, d), 7.0, dtype=torch.bfloat16, device="cuda")
    assert sk.kv4_attention(q, cache, table.cuda(), lens, off, out=out) is out
    assert torch.equal(out[:3], plain[:3]) and (out[3:] == 7).all() and (plain[3:] == 0).all()


def test_nan_and_infinity_reach_only_their_readers(sk):
    """A token with a NaN in its values spoils the rows that see it, and no other sequence, head or masked row."""
    g = torch.Generator().manual_seed(15)
    d, heads = 128, 2
    cache = sk.KV4Cache(8, heads, d, 16, 64)
    table = torch.tensor([[5, 1], [2, 7]], dtype=torch.int32).cuda()
    x = _bf16(g, 40, 2 * heads * d)
    x[9, 2 * d + 3] = float("nan")  # V of head 0, token 9 of sequence 0, first group
    lens, off = torch.tensor([20, 20], dtype=torch.int32).cuda(), torch.tensor([0, 20, 40], dtype=torch.int32).cuda()
    sk.kv4_append(x.cuda(), cache, table, lens, None, off)
    q = _bf16(g, 40, 4, d).cuda()
    out = sk.kv4_attention(q, cache, table, lens, off).cpu()
    spoiled = torch.isnan(out)
    assert spoiled[9:20, :2, :64].all()
    spoiled[9:20, :2, :64] = False
    assert not spoiled.any()
    only = sk.kv4_attention(q, cache, table, lens, off, window=5).cpu()
    assert torch.isnan(only[9:14, :2, :64]).all() and not torch.isnan(only[14:20]).any() and not torch.isnan(only[:9]).any()


@pytest.mark.parametrize("hq", [4, 12, 24])
def test_queries_that_are_no_numbers(sk, hq):
    """A NaN or an infinity in a query spoils its own row and head, and not a row that sees nothing."""
    g = torch.Generator().manual_seed(21)
    cache, table = _filled(sk, g, [40, 0, 9], 16, 2, 128, 64)
    lens = torch.tensor([40, 0, 9], dtype=torch.int32).cuda()
    q = _bf16(g, 3, hq, 128)
    good = sk.kv4_attention(q.cuda(), cache, table.cuda(), lens)
    q[0, 1, 5], q[2, hq - 1, 77], q[1, 0, 0] = float("nan"), float("inf"), float("nan")
    got = sk.kv4_attention(q.cuda(), cache, table.cuda(), lens)
    spoiled = torch.zeros(3, hq, dtype=torch.bool)
    spoiled[0, 1] = spoiled[2, hq - 1] = True
    assert torch.isnan(got[spoiled]).all() and torch.equal(got[~spoiled], good[~spoiled]) and (got[1] == 0).all()


@pytest.mark.parametrize("seqs", [257, 700, 4096])
def test_many_sequences(sk, seqs):
    """More sequences than a block has threads, most of them short or empty, one row each and several."""
    g = torch.Generator().manual_seed(seqs)
    lens = torch.randint(0, 20, (seqs,), generator=g)
    lens[seqs // 2] = 300
    page, hkv, hq, d = 32, 1, 2, 64
    width = 10
    table = torch.randint(0, 40, (seqs, width), generator=g).to(torch.int32)  # pages shared for reading
    cache = sk.KV4Cache(40, hkv, d, page, 32)
    fill = torch.arange(40, dtype=torch.int32).reshape(1, 40)
    off = torch.tensor([0, 40 * page], dtype=torch.int32).cuda()
    sk.kv4_append(_bf16(g, 40 * page, 2 * d).cuda(), cache, fill.cuda(), torch.tensor([40 * page], dtype=torch.int32).cuda(), None, off)
    k, v = ref.unpack(cache.pool, d, 32)
    news = torch.minimum(lens, torch.randint(0, 4, (seqs,), generator=g))
    for offs in (None, [0] + news.cumsum(0).tolist()):
        rows = seqs if offs is None else offs[-1]
        q = _bf16(g, rows, hq, d)
        got = sk.kv4_attention(q.cuda(), cache, table.cuda(), lens.to(torch.int32).cuda(), None if offs is None else torch.tensor(offs, dtype=torch.int32).cuda())
        want, slack = ref.attention(q, k, v, table.tolist(), lens.tolist(), offs, d ** -0.5, 0)
        _check(got, want, slack, f"{seqs} {offs is None}")
    assert sk._C.device_status() == 0


def test_bad_indices_are_reported_and_left_out(sk):
    """A page outside the pool, a length past the table, a position past the rotation's table, a slot past the pool."""
    g = torch.Generator().manual_seed(16)
    d = 128
    cache, table = _filled(sk, g, [40, 40, 40], 16, 2, d, 64)
    q = _bf16(g, 3, 4, d).cuda()
    lens = torch.tensor([40, 40, 40], dtype=torch.int32).cuda()
    good = sk.kv4_attention(q, cache, table.cuda(), lens)
    assert sk._C.device_status() == 0
    for bad in (-1, cache.pages, 1 << 30):
        broken = table.clone()
        broken[1, 1] = bad
        got = sk.kv4_attention(q, cache, broken.cuda(), lens)
        assert sk._C.device_status() == 5 and sk._C.device_status() == 0
        assert torch.equal(got[0], good[0]) and torch.equal(got[2], good[2]) and torch.isfinite(got).all()
        before = cache.pool.clone()
        sk.kv4_append(_bf16(g, 3, 8 * d).cuda(), cache, torch.full_like(broken, bad).cuda(), lens, None)
        assert sk._C.device_status() == 5 and torch.equal(before, cache.pool)
    for length in (49, -1, 1 << 30):
        got = sk.kv4_attention(q, cache, table.cuda(), torch.tensor([40, length, 40], dtype=torch.int32).cuda())
        assert sk._C.device_status() == 5
        assert torch.equal(got[0], good[0]) and torch.equal(got[2], good[2])
    before = cache.pool.clone()
    sk.kv4_append(_bf16(g, 3, 8 * d).cuda(), cache, table.cuda(), lens, sk.kv4.rotation_table(39, d))
    assert sk._C.device_status() == 5 and torch.equal(before, cache.pool)
    k, v = sk.kv4_read(cache, torch.tensor([-1, cache.pages * 16, 0]).cuda())
    assert sk._C.device_status() == 5 and (k[:2] == 0).all() and (v[:2] == 0).all()


def test_malformed_offsets_stay_inside_the_tensors(sk):
    """Offsets that run backwards or past the rows change only which rows are computed."""
    g = torch.Generator().manual_seed(17)
    cache, table = _filled(sk, g, [40, 40], 16, 2, 128, 64)
    lens = torch.tensor([40, 40], dtype=torch.int32).cuda()
    q = _bf16(g, 4, 4, 128).cuda()
    before = cache.pool.clone()
    for off in ([0, 3, 1], [0, 2, 900], [-5, 2, 4], [4, 4, 4], [3, 0, 0]):
        o = torch.tensor(off, dtype=torch.int32).cuda()
        assert torch.isfinite(sk.kv4_attention(q, cache, table.cuda(), lens, o)).all()
    assert torch.equal(before, cache.pool)
    sk._C.device_status()


def test_no_rows_and_no_sequences(sk):
    cache = sk.KV4Cache(1, 2, 128, 16, 64)
    table, lens = torch.zeros(0, 1, dtype=torch.int32).cuda(), torch.zeros(0, dtype=torch.int32).cuda()
    assert sk.kv4_attention(torch.zeros(0, 4, 128, dtype=torch.bfloat16).cuda(), cache, table, lens).shape == (0, 4, 128)
    assert sk.kv4_append(torch.zeros(0, 8 * 128, dtype=torch.bfloat16).cuda(), cache, table, lens, None).shape == (0, 4, 128)
    assert sk.kv4_read(cache, torch.zeros(0, dtype=torch.int64).cuda())[0].shape == (0, 2, 128)
    # rows, but no sequence that owns them
    off = torch.zeros(1, dtype=torch.int32).cuda()
    q = torch.ones(3, 4, 128, dtype=torch.bfloat16).cuda()
    assert (sk.kv4_attention(q, cache, table, lens, off) == 0).all()
    # a table of no pages: every length but 0 is past it
    none = torch.zeros(2, 0, dtype=torch.int32).cuda()
    assert (sk.kv4_attention(q[:2], cache, none, torch.zeros(2, dtype=torch.int32).cuda()) == 0).all()
    assert sk._C.device_status() == 0


def test_same_bits_every_run_and_on_any_stream(sk):
    g = torch.Generator().manual_seed(18)
    lens = [5000, 1, 777, 4000]
    cache, table = _filled(sk, g, lens, 64, 2, 128, 64)
    q, t, n = _bf16(g, 4, 8, 128).cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
    first = sk.kv4_attention(q, cache, t, n)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(sk.kv4_attention(q, cache, t, n))
    torch.cuda.synchronize()
    assert all(torch.equal(o, first) for o in outs)


def test_captured_graphs(sk):
    """Two captured graphs replayed in turn and at once; lengths that grow between replays are read on the device."""
    g = torch.Generator().manual_seed(19)
    d, hq, hkv = 128, 8, 2
    cache, table = _filled(sk, g, [900, 900], 64, hkv, d, 64)
    t = table.cuda()
    graphs = []
    for i in range(2):
        qkv = _bf16(g, 2, (hq + 2 * hkv) * d).cuda()
        lens = torch.tensor([1, 1], dtype=torch.int32).cuda()
        mine = sk.KV4Cache.from_pool(cache.pool.clone(), d, 64)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            sk.kv4_attention(sk.kv4_append(qkv, mine, t, lens, None), mine, t, lens)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = sk.kv4_attention(sk.kv4_append(qkv, mine, t, lens, None), mine, t, lens)
        graphs.append((graph, qkv, lens, mine, out))
    sides = [torch.cuda.Stream() for _ in range(2)]
    for step in ([10, 500], [11, 501], [900, 3]):
        want = []
        for graph, qkv, lens, mine, out in graphs:
            lens.copy_(torch.tensor(step, dtype=torch.int32))
            other = sk.KV4Cache.from_pool(mine.pool.clone(), d, 64)
            want.append(sk.kv4_attention(sk.kv4_append(qkv, other, t, lens, None), other, t, lens))
        torch.cuda.synchronize()
        for (graph, *_), s in zip(graphs, sides):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for (*_, out), w in zip(graphs, want):
            assert torch.equal(out, w)


def test_offsets_past_32_bits(sk):
    """A pool of more than 4 GiB: pages at its far end."""
    g = torch.Generator().manual_seed(20)
    d, hkv, page = 128, 8, 64
    pages = (5 << 30) // (hkv * page // 16 * sk._C.kv4_tile_bytes(d, 64))
    cache = sk.KV4Cache(pages, hkv, d, page, 64)
    small, table = _filled(sk, g, [150], page, hkv, d, 64)
    far = torch.tensor([[pages - 1, pages // 2, pages - 2]], dtype=torch.int32).cuda()
    for i, src in enumerate(table[0].tolist()):
        cache.pool[int(far[0, i])] = small.pool[src]
    q, lens = _bf16(g, 1, 32, d).cuda(), torch.tensor([150], dtype=torch.int32).cuda()
    assert torch.equal(sk.kv4_attention(q, cache, far, lens), sk.kv4_attention(q, small, table.cuda(), lens))
    slots = torch.tensor([int(far[0, 0]) * page + 5]).cuda()
    assert torch.equal(sk.kv4_read(cache, slots)[0], sk.kv4_read(small, torch.tensor([int(table[0, 0]) * page + 5]).cuda())[0])


def test_refusals(sk):
    cache = sk.KV4Cache(4, 2, 128, 16, 64)
    table, lens = torch.zeros(2, 2, dtype=torch.int32).cuda(), torch.ones(2, dtype=torch.int32).cuda()
    q = torch.zeros(2, 4, 128, dtype=torch.bfloat16).cuda()
    qkv = torch.zeros(2, 8 * 128, dtype=torch.bfloat16).cuda()
    for kw in (dict(head_dim=96), dict(group=16), dict(head_dim=64, group=128), dict(page_size=24), dict(page_size=2048), dict(pages=0), dict(kv_heads=0)):
        with pytest.raises(ValueError):
            sk.KV4Cache(**{**dict(pages=1, kv_heads=1), **kw})
    bad = [
        lambda: sk.KV4Cache.from_pool(cache.pool, 64, 64),
        lambda: sk.KV4Cache.from_pool(cache.pool[..., :-1], 128, 64),
        lambda: sk.kv4_attention(q.float(), cache, table, lens),
        lambda: sk.kv4_attention(q[..., :64], cache, table, lens),
        lambda: sk.kv4_attention(q[:, :3], cache, table, lens),
        lambda: sk.kv4_attention(q[:1], cache, table, lens),
        lambda: sk.kv4_attention(q, cache, table.long(), lens),
        lambda: sk.kv4_attention(q, cache, table, lens.long()),
        lambda: sk.kv4_attention(q, cache, table[:1], lens),
        lambda: sk.kv4_attention(q, cache, table.cpu(), lens),
        lambda: sk.kv4_attention(q, cache, table, lens, lens),
        lambda: sk.kv4_attention(q, cache, table, lens, window=-1),
        lambda: sk.kv4_attention(q, cache, table, lens, scale=float("nan")),
        lambda: sk.kv4_attention(q, cache, table, lens, out=q.float()),
        lambda: sk.kv4_attention(q.transpose(1, 2).contiguous().transpose(1, 2), cache, table, lens),
        lambda: sk.kv4_append(qkv.float(), cache, table, lens, None),
        lambda: sk.kv4_append(qkv[:, :-1], cache, table, lens, None),
        lambda: sk.kv4_append(qkv[:, : 3 * 128], cache, table, lens, None),
        lambda: sk.kv4_append(qkv[:1], cache, table, lens, None),
        lambda: sk.kv4_append(qkv, cache, table, lens, torch.zeros(4, 20).cuda()),
        lambda: sk.kv4_append(qkv, cache, table, lens, torch.zeros(4, 136).cuda()),
        lambda: sk.kv4_append(qkv, cache, table, lens, torch.zeros(4, 128).cuda().double()),
        lambda: sk.kv4_attention(q, cache, table, lens, out=q),
        lambda: sk.kv4_attention(q.repeat(2500, 1, 1)[:4097], cache, table[:1].repeat(4097, 1), lens[:1].repeat(4097)),
        lambda: sk.kv4_attention(q, cache, torch.zeros(2, (1 << 26) + 1, dtype=torch.int32).cuda(), lens),
        lambda: sk.kv4_read(cache, lens),
        lambda: sk.kv4_read(cache, torch.zeros(2, dtype=torch.int64)),
    ]
    for i, call in enumerate(bad):
        with pytest.raises((RuntimeError, ValueError)):
            call()
            raise AssertionError(f"call {i} was taken")
    assert sk._C.device_status() == 0


def test_zeroed_rest_without_offsets(sk):
    """The C entries asked to zero the rows behind the last sequence where every sequence has one row: there are none."""
    g = torch.Generator().manual_seed(21)
    cache, table = _filled(sk, g, [40, 3], 16, 2, 128, 64)
    table, lens = table.cuda(), torch.tensor([40, 3], dtype=torch.int32).cuda()
    q, out = _bf16(g, 2, 4, 128).cuda(), torch.full((2, 4, 128), 7.0, dtype=torch.bfloat16).cuda()
    want = sk.kv4_attention(q, cache, table, lens)
    nbytes = sk._C._kv4_workspace_bytes(2, 2, 4, 2, 128)
    ws, stream = torch.empty(nbytes, dtype=torch.uint8).cuda(), torch.cuda.current_stream().cuda_stream
    assert sk._C._spk_kv4_attention(q.data_ptr(), 512, cache.pool.data_ptr(), cache.pages, 16, 4, 2, 128, 64, table.data_ptr(), table.shape[1], lens.data_ptr(),
                                    None, 2, 2, 128 ** -0.5, 0, out.data_ptr(), 1, ws.data_ptr(), nbytes, stream) == 0
    assert torch.equal(out, want)
    qkv = _bf16(g, 2, 8 * 128).cuda()
    assert sk._C._spk_kv4_append(qkv.data_ptr(), 1024, cache.pool.data_ptr(), cache.pages, 16, 4, 2, 128, 64, table.data_ptr(), table.shape[1], lens.data_ptr(),
                                 None, 2, 2, None, 0, 0, out.data_ptr(), 1, stream) == 0
    assert torch.equal(out, qkv[:, :512].reshape(2, 4, 128))


def test_a_length_past_the_table_is_padding(sk):
    """A sequence that has outgrown its row of the table: nothing of it is written or read, the others are served."""
    g = torch.Generator().manual_seed(22)
    cache, table = _filled(sk, g, [48, 20], 16, 2, 128, 64)
    table, lens = table.cuda(), torch.tensor([49, 21], dtype=torch.int32).cuda()
    k0, v0 = ref.unpack(cache.pool, 128, 64)
    qkv = _bf16(g, 2, 8 * 128).cuda()
    q = sk.kv4_append(qkv, cache, table, lens, None)
    assert sk._C.device_status() == 5 and (q[0] == 0).all() and torch.equal(q[1], qkv[1, :512].reshape(4, 128))
    k, v = ref.unpack(cache.pool, 128, 64)
    full = table[0].tolist()
    assert torch.equal(k[full], k0[full]) and torch.equal(v[full], v0[full])
    assert not torch.equal(k[int(table[1, 1]), 4], k0[int(table[1, 1]), 4])
    out = sk.kv4_attention(q, cache, table, lens)
    assert sk._C.device_status() == 5 and (out[0] == 0).all()
    want, slack = ref.attention(q[1:], k, v, table[1:].tolist(), [21], None, 128 ** -0.5, 0)
    _check(out[1:], want, slack)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("more", [-24, -8, 8, -1])
def test_numbers_of_rotated_channels(sk, d, more):
    """Rotated channels just below half a head, above it, and one step short of all: q and the keys, to the roundings of a rotation
    in fp32 (2^-22 of the largest input) and, for the keys, of a code."""
    g = torch.Generator().manual_seed(d + more)
    hq, hkv, rows = 3, 2, 20
    rot = d - 8 if more == -1 else d // 2 + more
    cs = sk.kv4.rotation_table(64, rot, device="cpu")
    cache, table = sk.KV4Cache(3, hkv, d, 16, 32), torch.tensor([[2, 0, 1]], dtype=torch.int32).cuda()
    qkv = _bf16(g, rows, (hq + 2 * hkv) * d)
    lens, off = torch.tensor([37], dtype=torch.int32).cuda(), torch.tensor([0, rows], dtype=torch.int32).cuda()
    q = sk.kv4_append(qkv.cuda(), cache, table, lens, cs.cuda(), off).cpu().double()
    x = qkv.double().reshape(rows, -1, d)
    want = ref.rotate(x[:, : hq + hkv], cs[17:37])
    assert ((q - want[:, :hq]).abs() <= want[:, :hq].abs() * 2 ** -8 + 2.0 ** -22 * x.abs().amax()).all()
    pos = torch.arange(17, 37)
    k, v = (t.cpu().double() for t in sk.kv4_read(cache, (torch.tensor([2, 0, 1])[pos // 16] * 16 + pos % 16).cuda()))
    want_k, s, _ = ref.quantize(want[:, hq:], 32)
    assert ((k - want_k).abs() <= want_k.abs() * 2 ** -8 + s * (1 + 2 ** -7) + 15 * s * 2 ** -7).all()
    assert torch.equal(v, ref.quantize(x[:, hq + hkv:], 32)[0].to(torch.bfloat16).double())


def test_a_bad_index_does_not_hide_a_wait_that_gave_up(sk):
    """Both are reported, the wait first, whichever came first; and a split-K GEMM after them is right."""
    g = torch.Generator().manual_seed(23)
    cache, table = _filled(sk, g, [20], 16, 2, 128, 64)
    q, past = _bf16(g, 1, 4, 128).cuda(), torch.tensor([1 << 20], dtype=torch.int32).cuda()
    w = sk.W4Weight.quantize((torch.randn(4096, 256, generator=g) / 64).to(torch.bfloat16).cuda())
    a = _bf16(g, 1, 4096).cuda()
    want = sk.w4gemm(a, w)
    assert sk._C.device_status() == 0
    for first in (True, False):
        if first:
            sk.kv4_attention(q, cache, table.cuda(), past)
        sk._C.debug_expire_wait(4096)
        if not first:
            sk.kv4_attention(q, cache, table.cuda(), past)
        assert [sk._C.device_status() for _ in range(3)] == [3, 5, 0]
        assert torch.equal(sk.w4gemm(a, w), want)
