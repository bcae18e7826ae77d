"""The 4-bit K/V cache without a GPU: the C entry points refuse what they do not take, before any
launch; the oracle's format holds what it should."""

import ctypes as C

import numpy as np
import pytest

from llmnputest_amd import _lib, kv4
from oracle import kv4_oracle as ko

ERR_ARG, ERR_SHAPE, ERR_WS = -1, -2, -3
P = C.c_void_p(0x10000)      # aligned, never dereferenced
ODD = C.c_void_p(0x10008)
ODD4 = C.c_void_p(0x10004)


def cache(**kw):
    f = dict(pages=0x10000, page_stride=43008, table=0x10000, table_stride=16, n_pages=100, page_len=64,
             n_kv_heads=8, head_dim=64, n_seqs=4, table_len=16)
    f.update(kw)
    return _lib.Kv4(**f)


def call(name, *args):
    rc = getattr(_lib.lib(), name)(*args)
    return rc, _lib.lib().q4nx_last_error().decode()


def append(c, k=P, v=P, by=0, rows=4, row=512, head=64, seq=0, pos=P, cu=None, new=1):
    return call("q4nx_kv4_append", c, k, v, by, rows, row, head, seq, pos, cu, new, None)


def read(c, k=P, v=P, rows=4, pos=P, cu=None, new=1):
    return call("q4nx_kv4_read", c, k, v, 0, rows, pos, cu, new, None)


def attn(c, q=P, stride=2560, out=P, hq=40, cu=None, total=4, new=1, lens=P, most=1000, sel=None, n_sel=0,
         split=1, ws=None, n=0):
    return call("q4nx_kv4_attn", c, q, stride, out, None, hq, cu, total, new, lens, most, C.c_float(0.125),
                sel, n_sel, split, ws, n, None)


def select(c, q=P, stride=2560, hq=40, lens=P, most=1000, n_sel=8, first=1, last=1, sel=P, ws=P, n=1 << 20):
    return call("q4nx_kv4_select", c, q, stride, hq, lens, most, n_sel, first, last, sel, ws, n, None)


BAD_CACHES = [dict(pages=None), dict(table=None), dict(head_dim=96), dict(page_len=48), dict(page_len=16),
              dict(n_kv_heads=0), dict(n_kv_heads=1025), dict(n_pages=0), dict(n_seqs=0), dict(n_seqs=8193),
              dict(table_len=0), dict(table_len=17), dict(table_len=1 << 25, table_stride=1 << 25),
              dict(page_stride=43007), dict(page_stride=43000), dict(pages=0x10008), dict(head_dim=128)]


@pytest.mark.parametrize("bad", BAD_CACHES, ids=str)
def test_bad_caches_are_refused(bad):
    c = cache(**bad)
    for f in (append, read, attn, select):
        rc, msg = f(c)
        assert rc in (ERR_ARG, ERR_SHAPE) and "q4nx_kv4_" in msg, f
    for rc, _ in (call("q4nx_kv4_reserve", c, P, P, None, P, 1 << 20, None),
                  call("q4nx_kv4_fork", c, 0, 1, P, P, P, P, 1, None, P, 1 << 20, None),
                  call("q4nx_kv4_free", c, P, P, P, 1, None, None),
                  call("q4nx_kv4_compact", c, 0, 1, P, None, P, 1 << 20, None),
                  call("q4nx_kv4_copy_pages", c, 0, 1, P, P, 1, None)):
        assert rc in (ERR_ARG, ERR_SHAPE)
    assert _lib.lib().q4nx_kv4_attn_ws_bytes(c, 40, 0, 1, 1000, 0, 4) == 0
    assert _lib.lib().q4nx_kv4_select_ws_bytes(c, 1000) == 0
    assert _lib.lib().q4nx_kv4_pages_ws_bytes(c, 1) == 0


def test_null_cache_is_refused():
    for f in (append, read, attn, select):
        assert f(None)[0] == ERR_ARG


@pytest.mark.parametrize("kw,code", [(dict(k=None), ERR_ARG), (dict(v=ODD), ERR_ARG), (dict(pos=None), ERR_ARG),
                                     (dict(row=12), ERR_SHAPE), (dict(head=4), ERR_SHAPE),
                                     (dict(seq=-8), ERR_SHAPE), (dict(rows=0), ERR_SHAPE),
                                     (dict(by=2), ERR_SHAPE), (dict(new=0, cu=P), ERR_ARG),
                                     (dict(new=2), ERR_ARG), (dict(new=1 << 30, cu=P), ERR_SHAPE)], ids=str)
def test_append_refusals(kw, code):
    assert append(cache(), **kw)[0] == code


@pytest.mark.parametrize("kw,code", [(dict(k=None), ERR_ARG), (dict(v=ODD), ERR_ARG), (dict(rows=0), ERR_SHAPE),
                                     (dict(new=2), ERR_ARG)], ids=str)
def test_read_refusals(kw, code):
    assert read(cache(), **kw)[0] == code


@pytest.mark.parametrize("kw,code", [
    (dict(q=None), ERR_ARG), (dict(q=ODD), ERR_ARG), (dict(out=None), ERR_ARG), (dict(lens=None), ERR_ARG),
    (dict(hq=44), ERR_SHAPE), (dict(hq=136, stride=136 * 64), ERR_SHAPE), (dict(total=5), ERR_SHAPE),
    (dict(new=2), ERR_SHAPE), (dict(cu=P, total=0), ERR_SHAPE), (dict(cu=P, new=0), ERR_SHAPE),
    (dict(stride=2552), ERR_SHAPE), (dict(stride=2564), ERR_SHAPE), (dict(most=0), ERR_SHAPE),
    (dict(sel=P), ERR_ARG), (dict(n_sel=4), ERR_ARG), (dict(sel=P, n_sel=4, cu=P, new=2), ERR_SHAPE),
    (dict(split=-1), ERR_ARG), (dict(split=1025), ERR_ARG), (dict(split=2), ERR_WS),
    (dict(split=2, ws=P, n=1000), ERR_WS), (dict(out=ODD4), ERR_ARG),
    (dict(cu=P, total=1 << 25), ERR_SHAPE)], ids=str)
def test_attn_refusals(kw, code):
    assert attn(cache(), **kw)[0] == code


@pytest.mark.parametrize("kw,code", [
    (dict(q=None), ERR_ARG), (dict(q=ODD), ERR_ARG), (dict(sel=None), ERR_ARG), (dict(lens=None), ERR_ARG),
    (dict(hq=44), ERR_SHAPE), (dict(n_sel=0), ERR_ARG), (dict(n_sel=1), ERR_ARG), (dict(first=-1), ERR_ARG),
    (dict(stride=2552), ERR_SHAPE), (dict(most=0), ERR_SHAPE), (dict(ws=None), ERR_WS), (dict(n=70), ERR_WS)],
    ids=str)
def test_select_refusals(kw, code):
    assert select(cache(), **kw)[0] == code


def test_select_refuses_more_pages_than_it_holds():
    c = cache(table_len=20000, table_stride=20000)
    rc, msg = select(c, most=1 << 30)
    assert rc == ERR_SHAPE and "16384" in msg
    assert select(c, most=16385 * 64)[0] == ERR_SHAPE


def test_page_call_refusals():
    c = cache()
    big = 1 << 20
    assert call("q4nx_kv4_reserve", c, None, P, None, P, big, None)[0] == ERR_ARG
    assert call("q4nx_kv4_reserve", c, P, P, None, P, 64, None)[0] == ERR_WS
    assert call("q4nx_kv4_reserve", cache(n_seqs=8192, n_pages=1 << 20), P, P, None, P, big, None)[0] == ERR_SHAPE
    fork = lambda **k: call("q4nx_kv4_fork", c, *[{**dict(stride=43008 * 100, layers=2, lens=P, refs=P, src=P,  # noqa: E731
                            dst=P, n=2, status=None, ws=P, nb=big), **k}[x] for x in
                            ("stride", "layers", "lens", "refs", "src", "dst", "n", "status", "ws", "nb")], None)[0]
    assert fork(n=0) == ERR_SHAPE and fork(n=5) == ERR_SHAPE and fork(src=None) == ERR_ARG
    assert fork(stride=1000) == ERR_SHAPE and fork(layers=0) == ERR_SHAPE and fork(nb=10) == ERR_WS
    assert fork(stride=43008 * 100 + 8) == ERR_SHAPE
    assert call("q4nx_kv4_free", c, P, P, P, 5, None, None)[0] == ERR_SHAPE
    assert call("q4nx_kv4_free", c, P, None, P, 1, None, None)[0] == ERR_ARG
    assert call("q4nx_kv4_compact", c, 0, 1, None, None, P, big, None)[0] == ERR_ARG
    assert call("q4nx_kv4_compact", c, 0, 1, P, None, None, 0, None)[0] == ERR_WS
    assert call("q4nx_kv4_copy_pages", c, 0, 1, P, P, 0, None)[0] == ERR_SHAPE
    assert call("q4nx_kv4_copy_pages", c, 0, 1, None, P, 1, None)[0] == ERR_ARG


def test_python_refuses_before_the_library():
    with pytest.raises(ValueError, match="page"):
        kv4.page_bytes(48, 8, 64)
    with pytest.raises(ValueError, match="positive"):
        kv4.Kv4Cache(1, 0, 1, 64)
    import torch
    t = torch.zeros
    with pytest.raises(ValueError, match="GPU"):   # a cache lives on the device
        kv4.Kv4Cache.over(t((1, 4, 43008), dtype=torch.uint8), t((2, 2), dtype=torch.int32),
                          t(2, dtype=torch.int32), t(4, dtype=torch.int32))


def test_a_table_view_keeps_its_stride():
    """Rows of a wider table, a single row of any stride, and one row shown twice: its stride 0 has to
    reach the library, which refuses it (with the width in its place row 1 would be read behind row 0)."""
    import torch
    t = torch.zeros((6, 10), dtype=torch.int32)
    assert kv4._row_stride(t[1:5, :4]) == 10 and kv4._row_stride(t[::2]) == 20
    assert kv4._row_stride(t[2:3, :4]) == 4 and kv4._row_stride(t[:1].expand(1, 10)) == 10
    assert kv4._row_stride(t[:1].expand(3, 10)) == 0
    for f in (append, read, attn, select):
        assert f(cache(table_stride=0))[0] == ERR_SHAPE


def shares(lens, hkv, cap, line_groups, mean):
    """The parts that single tokens are cut into, as the kernel finds them from the lengths: a list of
    (item, part, parts, record) for the calls without n_split and with a counter for each item."""
    tiles = [max(1, -(-min(max(int(n), 0), cap) // 32)) for n in lens]
    total = sum(tiles) * hkv
    out = []
    if total <= 16384 or total <= mean * len(lens) * hkv:
        room = max(line_groups - len(lens) * hkv // 2, line_groups // 2)
        unit = min(max(-(-total // room), total // (32 * len(lens) * hkv), 8 if total < 1024 else 16), 128)
        at = 0
        for b, n in enumerate(tiles):
            for h in range(hkv):
                parts = -(-n // unit)
                out += [(b * hkv + h, p, parts, at + p) for p in range(parts)]
                at += parts
        return out
    unit, off = -(-total // line_groups), 0
    for b, n in enumerate(tiles):
        for h in range(hkv):
            first, last = off // unit, (off + n - 1) // unit
            out += [(b * hkv + h, g - first, last - first + 1, 2 * g + (g == first)) for g in range(first, last + 1)]
            off += n
    return out


@pytest.mark.parametrize("d,groups,mean", [(64, 768, 256), (128, 512, 64)])
def test_the_workspace_holds_every_share(d, groups, mean):
    """Wherever the lengths cut an item in parts, the call had to ask for a workspace, and its records lie
    within it, each written by one workgroup."""
    rng = np.random.default_rng(5)
    cases = [(1024, 8, 8), (2040, 8, 4), (512, 8, 16), (2048, 8, 2), (2048, 8, 1), (1, 1, 1), (1, 8, 17), (64, 8, 512),
             (3, 2, 9000), (1, 1, 20000), (256, 64, 9), (2048, 8, 100), (300, 8, 70), (100, 8, 300)]
    cases += [(int(rng.integers(1, 400)), int(rng.integers(1, 40)), int(rng.integers(1, 60))) for _ in range(60)]
    for n_seqs, hkv, tiles in cases:
        c = cache(n_seqs=n_seqs, n_kv_heads=hkv, head_dim=d, page_len=32, table_len=tiles, table_stride=tiles,
                  page_stride=1 << 24)
        group = int(rng.integers(1, 17))
        size = _lib.lib().q4nx_kv4_attn_ws_bytes(C.byref(c), group * hkv, 0, 1, 1 << 30, 0, 0)
        records = (size - 65536) // (-(-group // 4) * 4 * (d + 4) * 4) if size else 0
        if tiles <= 32 or (n_seqs * hkv >= 512 and tiles <= 64):
            assert size == 0   # one part each
            continue
        for lens in ([tiles * 32] * n_seqs, [0] * n_seqs, rng.integers(0, tiles * 32 + 40, n_seqs)):
            all_ = shares(lens, hkv, tiles * 32, groups, mean)
            cut = [x for x in all_ if x[2] > 1]
            items, most = n_seqs * hkv, n_seqs * hkv * tiles
            grid = items + max(min(most // 8, groups), min(most, mean * items) // 128)   # as launched
            line = sum(max(1, -(-min(int(n), tiles * 32) // 32)) for n in lens) * hkv
            if not (line > 16384 and line > mean * items):
                assert len(all_) <= min(grid, items * -(-tiles // 8)) or most > 16384 and len(all_) <= max(grid, groups)
            if not size and 5 * n_seqs * hkv * -(-group // 4) * 16 * (d + 4) > 192 << 20:
                continue   # records of thousands of items would not fit: one part each
            assert not cut or size, (n_seqs, hkv, tiles)
            places = [x[3] for x in cut]
            assert len(set(places)) == len(places) and max(places, default=-1) < records
            assert max((x[0] for x in cut), default=0) * 4 < 65536


def test_page_bytes():
    f = _lib.lib().q4nx_kv4_page_bytes
    assert f(64, 8, 64) == 8 * (2 * 2560 + 256) and f(32, 1, 128) == 5120 + 512
    assert f(16, 8, 64) == f(64, 0, 64) == f(64, 8, 80) == 0


# ------------------------------------------------------------------ the oracle's own format

@pytest.mark.parametrize("d", [64, 128])
def test_format_places_are_a_partition(d):
    """Every nibble of a tile's code bytes belongs to one position and channel of K or of V."""
    seen = np.zeros((32 * d, 2), int)
    for byte, nib in ko.places(d):
        np.add.at(seen, (byte, nib), 1)
    assert (seen == 1).all()


@pytest.mark.parametrize("d", [64, 128])
def test_format_holds_rows_to_half_a_step(d):
    """|x - (d code + m)| is at most half a step, and what rounding d to bf16 (2^-8) leaves out of the
    top: 15 d 2^-8 in all."""
    rng = np.random.default_rng(d)
    x = ko.bf16_f32(ko.bf16_bits(rng.standard_normal((33, 2, d)).astype(np.float32) * 3))
    pages = ko.Pages(np.zeros((2, 2 * (2 * 40 * d + 4 * d)), np.uint8), 2, d, 64)
    table = np.array([[1]], np.int32)
    pages.append(table, [5], [range(33)], x, -x)
    for i in range(33):
        for h in range(2):
            for got, want in zip(pages.values(1, h, 5 + i), (x[i, h], -x[i, h])):
                step = np.repeat((want.reshape(-1, 32).max(-1) - want.reshape(-1, 32).min(-1)) / 15, 32)
                assert (np.abs(got - want) <= step * (0.5 + 2.0 ** -7 + 15 * 2.0 ** -8)).all()
    assert not pages.pool[0].any()


def test_quant_rules():
    x = np.zeros((4, 32), np.float32)
    x[0, 3] = np.nan
    x[1, 7] = np.inf
    x[2, 0], x[2, 1] = 3e38, -3e38       # the range overflows
    x[3] = 1.5                           # no range: the value itself
    codes, d, m = ko.quant(x)
    assert (d[:3] == 0x7FC0).all() and (m[:3] == 0x7FC0).all() and not codes.any()
    assert d[3, 0] == 0 and ko.bf16_f32(m[3, 0]) == 1.5
    y = np.arange(32, dtype=np.float32)  # ties go to even: d = bf16(31 / 15)
    codes, d, _ = ko.quant(y[None])
    q = y / ko.bf16_f32(d[0, 0])
    assert (codes[0] == np.minimum(np.rint(q), 15)).all()


def test_book_fork_and_compact():
    b = ko.Book(4, 4, 10, 32)
    assert b.reserve([70, 10, 0, 0]) == 0 and b.table[0, :3].tolist() == [0, 1, 2] and b.table[1, 0] == 3
    b.lens[:] = [70, 10, 0, 0]
    assert b.fork([0, 1, 0], [2, 2, 9]) == 2
    assert b.table[2].tolist() == [0, 1, 4, -1] and b.refs[:5].tolist() == [2, 2, 1, 1, 1]
    assert b.free([0]) == 0 and b.refs[:5].tolist() == [1, 1, 0, 1, 1]
    assert b.compact() == 4 and b.table[2].tolist() == [0, 1, 2, -1] and b.moves[-1] == (4, 2)
