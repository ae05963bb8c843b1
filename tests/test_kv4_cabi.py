"""Without a GPU: what the C entry points of the 4-bit cache and the residual norm refuse before they touch CUDA, with the
status and a message that names the argument; and the bytes of a tile."""

import ctypes
import os

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
i, p, ll, f = ctypes.c_int, ctypes.c_void_p, ctypes.c_longlong, ctypes.c_float


@pytest.fixture(scope="module")
def lib():
    lib = ctypes.CDLL(os.path.join(ROOT, "5090-blackwell-kernels_b200", "lib", "libspark_b200.so"))
    lib.spk_last_error.restype = ctypes.c_char_p
    lib.spk_kv4_attention_workspace.restype = ll
    lib.spk_kv4_append.argtypes = [p, ll, p, i, i, i, i, i, i, p, i, p, p, i, i, p, i, i, p, i, p]
    lib.spk_kv4_read.argtypes = [p, i, i, i, i, i, p, i, p, p, p]
    lib.spk_kv4_attention.argtypes = [p, ll, p, i, i, i, i, i, i, p, i, p, p, i, i, f, i, p, i, p, ll, p]
    lib.spk_add_rmsnorm.argtypes = [p, ll, p, ll, p, p, p, ll, f, f, p, p, i, i, p]
    return lib


@pytest.fixture(scope="module")
def at():
    buf = ctypes.create_string_buffer(256)
    base = ctypes.addressof(buf)
    yield lambda k: base + (-base) % 16 + 16 * k
    del buf


def _refused(lib, rc, word):
    assert rc == 1 and word in lib.spk_last_error().decode(), (rc, lib.spk_last_error())


def test_tile_bytes(lib):
    assert [lib.spk_kv4_tile_bytes(d, g) for d, g in ((64, 32), (64, 64), (128, 32), (128, 64), (128, 128))] == [1280, 1152, 2560, 2304, 2176]
    assert [lib.spk_kv4_tile_bytes(d, g) for d, g in ((64, 128), (96, 32), (128, 16), (0, 0), (256, 64))] == [0] * 5


def test_attention(lib, at):
    def call(**kw):
        a = dict(q=at(0), stride=512, pool=at(1), pages=4, page=16, hq=4, hkv=2, d=128, g=64, table=at(2), width=2, lens=at(3), off=None, seqs=2, rows=2,
                 scale=0.1, window=0, out=at(4), rest=0, ws=at(5), wsb=1 << 40, stream=None)
        a.update(kw)
        return lib.spk_kv4_attention(*a.values())

    for kw, word in ((dict(pool=None), "pool"), (dict(pool=at(1) + 8), "pool"), (dict(d=96), "head_dim"), (dict(g=48), "group"), (dict(d=64, g=128), "group"),
                     (dict(page=24), "page_size"), (dict(page=0), "page_size"), (dict(page=2048), "page_size"), (dict(pages=0), "page"), (dict(hkv=0), "KV heads"),
                     (dict(seqs=4097, rows=4097), "4096"), (dict(seqs=-1), "sequences"), (dict(rows=3), "q_offsets"), (dict(width=1 << 27), "2^30"),
                     (dict(lens=None), "lengths"), (dict(table=None), "page table"), (dict(hq=3), "q_heads"), (dict(window=-1), "window"),
                     (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(q=None), "q and out"), (dict(out=at(0)), "q and out"),
                     (dict(out=at(4) + 2), "q and out"), (dict(stride=511), "rows of q"), (dict(stride=504), "rows of q"), (dict(ws=None), "workspace"),
                     (dict(wsb=16), "workspace")):
        _refused(lib, call(**kw), word)
    assert call(seqs=0, rows=0) == 0  # nothing to do: nothing touched


def test_append_and_read(lib, at):
    def call(**kw):
        a = dict(qkv=at(0), stride=1024, pool=at(1), pages=4, page=16, hq=4, hkv=2, d=128, g=64, table=at(2), width=2, lens=at(3), off=None, seqs=2, rows=2,
                 cs=at(6), positions=8, rot=128, q=at(4), rest=0, stream=None)
        a.update(kw)
        return lib.spk_kv4_append(*a.values())

    for kw, word in ((dict(pool=None), "pool"), (dict(d=80), "head_dim"), (dict(rot=136), "rotated"), (dict(rot=20), "rotated"), (dict(positions=0), "rotation"),
                     (dict(cs=None), "null"), (dict(cs=at(6) + 4), "aligned"), (dict(qkv=None), "null"), (dict(q=None), "null"), (dict(q=at(0)), "memory"),
                     (dict(stride=1016), "apart"), (dict(stride=1028), "apart"), (dict(hq=-1), "q_heads"), (dict(rows=3), "q_offsets")):
        _refused(lib, call(**kw), word)
    assert call(seqs=0, rows=0) == 0
    _refused(lib, lib.spk_kv4_read(at(1), 4, 16, 2, 128, 64, None, 3, at(2), at(3), None), "null")
    _refused(lib, lib.spk_kv4_read(at(1), 4, 16, 2, 128, 64, at(0), -1, at(2), at(3), None), "slots")
    assert lib.spk_kv4_read(at(1), 4, 16, 2, 128, 64, None, 0, None, None, None) == 0


def test_norm(lib, at):
    def call(**kw):
        a = dict(x=at(0), xs=64, y=at(1), ys=64, gain=at(2), post=None, gate=None, gs=0, scale=1.0, eps=1e-5, r=at(3), h=at(4), rows=2, hidden=64, stream=None)
        a.update(kw)
        return lib.spk_add_rmsnorm(*a.values())

    for kw, word in ((dict(hidden=60), "hidden"), (dict(hidden=0), "hidden"), (dict(hidden=65544), "hidden"), (dict(rows=-1), "hidden"), (dict(eps=-1.0), "eps"),
                     (dict(eps=float("nan")), "eps"), (dict(x=None), "need y"), (dict(y=None, scale=0.5), "need y"), (dict(y=None, post=at(2)), "need y"),
                     (dict(r=None), "goes with"), (dict(h=None), "goes with"), (dict(gain=None), "goes with"), (dict(y=None, gain=None, h=None), "goes with"),
                     (dict(x=at(0) + 2), "aligned"), (dict(xs=68), "strides"), (dict(gs=-8), "strides")):
        _refused(lib, call(**kw), word)
    assert call(rows=0) == 0


def test_outputs_in_the_inputs_memory(lib, at):
    """An output that begins, ends or lies inside what the input's rows span."""
    buf = ctypes.create_string_buffer(16384)
    base = ctypes.addressof(buf)
    base += -base % 16
    for out in (base + 16, base + 1024 - 16, base + 2032):  # q: two rows of 1 KiB at base + 1024
        rc = lib.spk_kv4_attention(base + 1024, 512, at(1), 4, 16, 4, 2, 128, 64, at(2), 2, at(3), None, 2, 2, 0.1, 0, out, 0, at(5), 1 << 40, None)
        _refused(lib, rc, "out must not be in q's memory")
    for out in (base + 16, base + 2048 + 16, base + 2048 + 4080):  # qkv: two rows of 2 KiB at base + 2048
        rc = lib.spk_kv4_append(base + 2048, 1024, at(1), 4, 16, 4, 2, 128, 64, at(2), 2, at(3), None, 2, 2, at(6), 8, 128, out, 0, None)
        _refused(lib, rc, "q_out must not be in qkv's memory")


def test_norm_in_place_needs_contiguous_rows(lib, at):
    rc = lib.spk_add_rmsnorm(at(0), 72, at(1), 64, at(2), None, None, 0, 1.0, 1e-5, at(0), at(4), 2, 64, None)
    _refused(lib, rc, "r may be x")


def test_norm_outputs_in_the_inputs_memory(lib, at):
    """r or h anywhere in what x, y, a gate or the gains span, or in each other; in the place of one with contiguous rows they
    are not refused (without a GPU the call then ends at the device)."""
    buf = ctypes.create_string_buffer(16384)
    base = ctypes.addressof(buf)
    base += -base % 16
    place = {name: base + 1200 * i for i, name in enumerate(("x", "y", "gain", "post", "gate", "r", "h"), 1)}

    def call(xs=64, ys=64, gs=64, rows=2, **kw):
        a = place | kw
        return lib.spk_add_rmsnorm(a["x"], xs, a["y"], ys, a["gain"], a["post"], a["gate"], gs, 1.0, 1e-5, a["r"], a["h"], rows, 64, None)

    for out in ("r", "h"):
        for name, word in (("x", "of x"), ("y", "of y"), ("gain", "of the gain"), ("post", "of post_gain"), ("gate", "of the gate")):
            size = 128 if name in ("gain", "post") else 256
            for shift in (16 - 256, -128, 16, size - 16):
                _refused(lib, call(**{out: place[name] + shift}), word)
        _refused(lib, call(**{out: place["gain"]}), "of the gain")
        _refused(lib, call(**{out: place["y"]}, ys=72), "of y")
        _refused(lib, call(**{out: place["y"]}, ys=0), "of y")
        _refused(lib, call(**{out: place["gate"]}, gs=0), "of the gate")
        _refused(lib, call(**{out: place["gate"] + 112}, gs=0), "of the gate")
        for name in ("x", "y", "gate"):
            assert call(**{out: place[name]}) != 1, (out, name, lib.spk_last_error())
        assert call(**{out: place["y"]}, ys=72, rows=1) != 1
        assert call(**{out: place["gate"] + 128}, gs=0) != 1  # behind the one row that there is
    _refused(lib, call(h=place["x"], xs=72), "of x")
    _refused(lib, call(h=place["r"]), "share")
    _refused(lib, call(h=place["r"] + 240), "share")


def test_norm_without_y_does_not_look_at_r(lib, at):
    """r is not written then, wherever it points."""
    buf = ctypes.create_string_buffer(4096)
    base = ctypes.addressof(buf)
    base += -base % 16
    for r in (base, base + 16, base + 1024, base + 2048 + 16):
        assert lib.spk_add_rmsnorm(base, 64, None, 0, base + 1024, None, None, 0, 1.0, 1e-5, r, base + 2048, 2, 64, None) != 1, r - base
