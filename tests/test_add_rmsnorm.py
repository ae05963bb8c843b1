"""The residual norm against its definition in 64 bits. Tolerance: r is one rounding of a sum that fp32 holds to a few
2^-24, so half a step of bf16 (2^-8 of it) plus 2^-21 of the summands; h is a function of the r that was returned, again half a
step, plus 2^-18 for the sums in fp32."""

import pytest
import torch

pytestmark = pytest.mark.gpu
F64 = torch.float64


def _norm(v, eps):
    return v / (v.square().mean(-1, keepdim=True) + eps).sqrt()


def _check(x, y, gain, eps, post, gate, scale, r, h):
    d = lambda t: t.cpu().to(F64)  # noqa: E731
    xd = d(x)
    if y is not None:
        z = d(y) if post is None else _norm(d(y), eps) * d(post)
        z = z if gate is None else z * d(gate)
        want = scale * xd + z
        assert ((d(r) - want).abs() <= want.abs() * 2 ** -8 + 2.0 ** -21 * (abs(scale) * xd.abs() + z.abs()) + 1e-38).all()
    if gain is not None:
        want = _norm(d(r), eps) * d(gain)
        assert ((d(h) - want).abs() <= want.abs() * (2 ** -8 + 2.0 ** -18) + 1e-38).all()


def _bf16(g, *shape):
    return torch.randn(shape, generator=g).to(torch.bfloat16).cuda()


@pytest.mark.parametrize("hidden", [8, 64, 264, 1000, 4096, 5120, 8200, 16384, 20000, 65536])
@pytest.mark.parametrize("rows", [1, 3, 150])
@pytest.mark.parametrize("form", ["plain", "post", "channel", "row", "all"])
def test_against_64_bits(sk, rows, hidden, form):
    g = torch.Generator().manual_seed(hidden + rows)
    x, y, gain = 4 * _bf16(g, rows, hidden), _bf16(g, rows, hidden), _bf16(g, hidden)
    post = _bf16(g, hidden) if form in ("post", "all") else None
    gate = _bf16(g, hidden) if form == "channel" else _bf16(g, rows, hidden) if form in ("row", "all") else None
    scale = 0.7071 if form == "all" else 1.0
    r, h = sk.add_rmsnorm(x, y, gain, eps=1e-6, post_gain=post, gate=gate, residual_scale=scale)
    _check(x, y, gain, 1e-6, post, gate, scale, r, h)


def test_partial_forms_strides_and_many_rows(sk):
    g = torch.Generator().manual_seed(1)
    wide = _bf16(g, 700, 3 * 1024)
    x, y, gain = wide[:, :1024], wide[:, 1024:2048], _bf16(g, 1024)
    r, h = sk.add_rmsnorm(x, y, gain)
    _check(x, y, gain, 1e-5, None, None, 1.0, r, h)
    r2, h2 = sk.add_rmsnorm(x.contiguous(), y.contiguous(), gain)
    assert torch.equal(r, r2) and torch.equal(h, h2)
    r3, none = sk.add_rmsnorm(x, y)
    assert none is None and torch.equal(r3, r)
    same, h4 = sk.add_rmsnorm(x, gain=gain)
    assert same is x
    _check(x, None, gain, 1e-5, None, None, 1.0, x, h4)
    gate = _bf16(g, 1, 1024)
    a = sk.add_rmsnorm(x, y, gain, gate=gate.expand(700, 1024))
    b = sk.add_rmsnorm(x, y, gain, gate=gate[0])
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert sk.add_rmsnorm(x[:0], y[:0], gain)[1].shape == (0, 1024)


def test_extremes(sk):
    """Zero rows (eps alone), tiny and huge values, rows with a NaN or an infinity stay by themselves."""
    g = torch.Generator().manual_seed(2)
    x, y, gain = _bf16(g, 6, 512), _bf16(g, 6, 512), _bf16(g, 512)
    x[0] = y[0] = 0
    x[1], y[1] = 1e-30 * x[1], 1e-30 * y[1]
    x[2], y[2] = 1e15 * x[2], 1e15 * y[2]
    x[3, 5] = float("nan")
    y[4, 7] = float("inf")
    r, h = sk.add_rmsnorm(x, y, gain, eps=1e-5)
    keep = [0, 1, 2, 5]
    _check(x[keep], y[keep], gain, 1e-5, None, None, 1.0, r[keep], h[keep])
    assert (h[0] == 0).all() and torch.isnan(h[3]).all() and torch.isnan(r[3, 5]) and torch.isfinite(r[3, :5]).all()
    assert torch.isinf(r[4, 7]) and not torch.isfinite(h[4, 7])


def test_captured(sk):
    g = torch.Generator().manual_seed(3)
    x, y, gain = _bf16(g, 33, 2048), _bf16(g, 33, 2048), _bf16(g, 2048)
    want = sk.add_rmsnorm(x, y, gain)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = sk.add_rmsnorm(x, y, gain)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_refusals(sk):
    x = torch.zeros(4, 64, dtype=torch.bfloat16).cuda()
    gain = torch.ones(64, dtype=torch.bfloat16).cuda()
    for call in (
        lambda: sk.add_rmsnorm(x),
        lambda: sk.add_rmsnorm(x.float(), x, gain),
        lambda: sk.add_rmsnorm(x, x.float(), gain),
        lambda: sk.add_rmsnorm(x, x[:3], gain),
        lambda: sk.add_rmsnorm(x, x, gain[:32]),
        lambda: sk.add_rmsnorm(x, x, gain.float()),
        lambda: sk.add_rmsnorm(x[:, :60], x[:, :60], gain[:60]),
        lambda: sk.add_rmsnorm(x, gain=gain, post_gain=gain),
        lambda: sk.add_rmsnorm(x, gain=gain, residual_scale=0.5),
        lambda: sk.add_rmsnorm(x, x, gain, gate=x[:2]),
        lambda: sk.add_rmsnorm(x, x, gain, eps=-1.0),
        lambda: sk.add_rmsnorm(x.cpu(), x, gain),
        lambda: sk.add_rmsnorm(x.t(), x.t(), gain),
        lambda: sk.add_rmsnorm(x[:, 4:60], x[:, 4:60], gain[:56]),
    ):
        with pytest.raises((RuntimeError, ValueError)):
            call()


@pytest.mark.parametrize("rows,hidden", [(3, 4096), (700, 264), (400, 8200), (3, 40000)])
def test_outputs_in_the_place_of_inputs(sk, rows, hidden):
    """The C entry with r and h in the place of x, y or a gate with rows: the same bits as beside them."""
    g = torch.Generator().manual_seed(4)
    x, y, gate, gain, post = _bf16(g, rows, hidden), _bf16(g, rows, hidden), _bf16(g, rows, hidden), _bf16(g, hidden), _bf16(g, hidden)
    want = sk.add_rmsnorm(x, y, gain, post_gain=post, gate=gate, residual_scale=0.5)
    stream = torch.cuda.current_stream().cuda_stream
    for r_in, h_in in (("x", None), ("y", "x"), ("gate", "y"), (None, "gate")):
        t = {"x": x.clone(), "y": y.clone(), "gate": gate.clone(), None: None}
        r, h = (torch.empty_like(x) if name is None else t[name] for name in (r_in, h_in))
        assert sk._C._spk_add_rmsnorm(t["x"].data_ptr(), hidden, t["y"].data_ptr(), hidden, gain.data_ptr(), post.data_ptr(), t["gate"].data_ptr(), hidden,
                                      0.5, 1e-5, r.data_ptr(), h.data_ptr(), rows, hidden, stream) == 0
        assert torch.equal(r, want[0]) and torch.equal(h, want[1]), (r_in, h_in)


@pytest.mark.parametrize("hidden", [8, 1024, 1032, 2040, 2048, 2056, 5120, 8184, 8192, 8200, 20000, 32768, 32776, 65536])
@pytest.mark.parametrize("more", [0, 1, 400])
@pytest.mark.parametrize("form", ["plain", "all", "partial"])
def test_many_rows_against_64_bits(sk, hidden, more, form):
    """From two rows an SM up other blocks are launched, by the number of channels: every one at a full size, the next larger and a last
    piece that is not full, with the last count of rows of the other launch and the first of this."""
    rows = 2 * torch.cuda.get_device_properties(0).multi_processor_count + more
    g = torch.Generator().manual_seed(hidden + rows)
    x, y, gain = 4 * _bf16(g, rows, hidden), _bf16(g, rows, hidden), _bf16(g, hidden)
    if form == "partial":
        r, h = sk.add_rmsnorm(x, gain=gain, eps=1e-6)
        assert r is x
        _check(x, None, gain, 1e-6, None, None, 1.0, x, h)
        r, h = sk.add_rmsnorm(x, y, post_gain=gain)
        assert h is None
        return _check(x, y, None, 1e-5, gain, None, 1.0, r, None)
    post = _bf16(g, hidden) if form == "all" else None
    gate = _bf16(g, rows, hidden) if form == "all" else None
    scale = 0.7071 if form == "all" else 1.0
    r, h = sk.add_rmsnorm(x, y, gain, eps=1e-6, post_gain=post, gate=gate, residual_scale=scale)
    _check(x, y, gain, 1e-6, post, gate, scale, r, h)
