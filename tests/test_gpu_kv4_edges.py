"""Edges of the paged 4-bit K/V cache: infinities in a query, counts past one wave, lengths of zero,
positions at the ends of 32 bits, strides that say nothing."""

import numpy as np
import pytest
import torch

from llmnputest_amd import kv4
from oracle import kv4_oracle as ko
from tests.test_gpu_kv4 import Case, bf16, check, ints, up

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ selection

def signed_pages(dev, d, page, n, infinite, ch, hkv=1):
    """n pages whose channel `ch` of K is positive in the pages `infinite` and negative in the others."""
    x = Case(dev, 50, hkv, d, page, [n * page])
    k, v = x.rows(n * page), x.rows(n * page)
    k[..., ch] = -bf16(1 + np.abs(k[..., ch]))
    for p in infinite:
        k[p * page:(p + 1) * page, :, ch] *= -1
    x.c.append(0, up(k, dev), up(v, dev), ints([0], dev), ints([0, n * page], dev))
    x.o.append(x.table, [0], [range(n * page)], k, v)
    return x


@pytest.mark.parametrize("d,page", [(64, 32), (128, 64)])
@pytest.mark.parametrize("infinite", [[4, 9], [4], [1, 2, 3, 5, 8, 12], [0, 13], list(range(14)), []], ids=str)
@pytest.mark.parametrize("n_sel,first,last", [(4, 1, 1), (3, 0, 1), (2, 0, 0), (6, 3, 1), (2, 1, 1)])
def test_select_with_an_infinity_in_q(dev, d, page, infinite, n_sel, first, last):
    """Scores of +inf and -inf: the pages always read are there, then the infinite ones, the lowest first,
    and every entry is written, however many of them the list holds."""
    x = signed_pages(dev, d, page, 14, infinite, 5)
    q = x.q(1, 3)
    q[0, 1, 5] = np.inf
    out = torch.full((1, 1, n_sel), -77, dtype=torch.int32, device=dev)
    x.c.select(0, up(q, dev), ints([14 * page], dev), n_sel, first, last, out=out)
    want = ko.select(x.o, x.table[0], q[0].astype(np.float64), 14 * page, n_sel, first, last)
    assert np.array_equal(out[0].cpu().numpy(), want)


def test_select_with_infinities_of_both_signs(dev):
    """-inf in q, and +inf in one channel against -inf in another (scores that are NaN): as many lists as
    there are kv heads, each with its own."""
    x = signed_pages(dev, 64, 32, 20, [2, 7, 11], 40, hkv=2)
    q = x.q(1, 4)
    q[0, 0, 40], q[0, 3, 40], q[0, 3, 41] = -np.inf, np.inf, -np.inf
    for n_sel, first, last in ((5, 1, 1), (3, 1, 1), (17, 2, 3), (19, 0, 0)):
        with np.errstate(invalid="ignore"):
            want = ko.select(x.o, x.table[0], q[0].astype(np.float64), 640, n_sel, first, last)
        got = x.c.select(0, up(q, dev), ints([640], dev), n_sel, first, last)
        assert np.array_equal(got[0].cpu().numpy(), want), n_sel


# ------------------------------------------------------------------ bookkeeping

@pytest.mark.parametrize("n_seqs,n_pages", [(700, 1000), (3000, 20000), (65, 400)])
def test_reserve_counts_what_every_wave_refuses(dev, n_seqs, n_pages):
    """Hundreds of sequences that want more than their row holds, in every wave of the launch and in more
    than one round of it: `status` counts each."""
    rng = np.random.default_rng(n_seqs)
    for turn in range(6):
        c = kv4.Kv4Cache(1, n_pages, n_seqs, 4 * 32, n_kv_heads=1, page_len=32, device=dev)
        book = ko.Book(n_seqs, 4, n_pages, 32)
        want = rng.integers(0, 4 * 32 + 1, n_seqs)
        over = rng.random(n_seqs) < 0.5
        over[64:] |= turn == 0          # all of them but the first wave's
        want[over] += 4 * 32 + 1
        c.reserve(want.tolist())
        bad = book.reserve(want)
        assert int(c.status) == bad >= over.sum(), turn
        assert np.array_equal(c.table.cpu().numpy(), book.table)
        assert np.array_equal(c.refs.cpu().numpy(), book.refs)


def test_fork_of_a_source_without_its_pages(dev):
    """A source's length past the pages it has, a multiple of the page among them, is not done and changes
    nothing; at its last page it is done; a length of zero shares nothing."""
    for extra, done in ((0, True), (1, False), (31, False), (32, False), (64, False), (-1, True), (-64, True)):
        c = kv4.Kv4Cache(1, 9, 3, 6 * 32, n_kv_heads=1, page_len=32, device=dev)
        book = ko.Book(3, 6, 9, 32)
        c.reserve([64, 0, 20])
        book.reserve([64, 0, 20])
        book.lens[:] = [64 + extra, 0, 20]
        c.lens.copy_(torch.from_numpy(book.lens))
        c.fork([0, 2], [1, 1])       # the second pair's dst is taken either way
        assert book.fork([0, 2], [1, 1]) == 2 - done
        assert int(c.status) == 2 - done, extra
        assert np.array_equal(c.table.cpu().numpy(), book.table), extra
        assert np.array_equal(c.refs.cpu().numpy(), book.refs), extra
        assert np.array_equal(c.lens.cpu().numpy(), book.lens), extra
        assert (c.table[1, 0] >= 0).item() == (done and extra > -64)


def test_fork_of_a_row_that_names_no_page(dev):
    """The last full page's entry lies outside the pool: not done, and no entry of it is handed on."""
    c = kv4.Kv4Cache(1, 9, 2, 6 * 32, n_kv_heads=1, page_len=32, device=dev)
    c.reserve([64, 0])
    c.table[0, 1] = 1 << 20
    c.lens.copy_(ints([64, 0], dev))
    c.fork([0], [1])
    assert int(c.status) == 1 and (c.table[1] == -1).all() and c.lens.tolist() == [64, 0]
    assert c.refs.tolist() == [1, 1] + [0] * 7


# ------------------------------------------------------------------ arguments

def test_max_len_of_zero_reads_nothing(dev):
    """max_len=0 is a bound like any other: zeros, no pages, and rows behind the last sequence as they were."""
    x = Case(dev, 51, 2, 64, 32, [100, 70])
    x.fill([100, 70])
    lens, q = ints([100, 70], dev), up(x.q(2, 6), dev)
    out = torch.full_like(q, 3.0)
    got, got32 = x.c.attn(0, q, lens, max_len=0, out=out, want_f32=True)
    assert got is out and not got.any() and not got32.any()
    assert not x.c.attn(0, q, lens, max_len=0, n_split=4).any()
    block = up(x.q(40, 6), dev)
    out = torch.full_like(block, 3.0)
    for n_split in (0, 3):
        x.c.attn(0, block, lens, cu=ints([0, 30, 33], dev), max_len=0, out=out.fill_(3.0), n_split=n_split)
        assert not out[:33].any() and (out[33:] == 3).all()
    sel = x.c.select(0, q, lens, n_sel=3, max_len=0)
    assert (sel == -1).all() and not x.c.attn(0, q, lens, sel=sel).any()
    assert lens.tolist() == [100, 70]
    assert x.c.attn(0, q, lens, max_len=1).any()
    from llmnputest_amd import ops
    for call in (lambda: x.c.attn(0, q, lens, max_len=-1), lambda: x.c.select(0, q, lens, n_sel=3, max_len=-1)):
        with pytest.raises(ops._lib.Q4NXError, match="max_len"):
            call()


def test_a_block_of_more_than_a_million_tokens(dev):
    """All but the last rows stand before the cache's first position and see nothing."""
    x = Case(dev, 55, 1, 64, 64, [70])
    x.fill([70])
    n = (1 << 20) + 77
    q = x.q(100, 1)
    many = torch.ones((n, 1, 64), dtype=torch.bfloat16, device=dev)
    many[-100:] = up(q, dev)
    got, got32 = x.c.attn(0, many, ints([70], dev), cu=ints([0, n], dev), want_f32=True)
    assert not got[:-70].any() and not got32[:-70].any()
    check(got[-70:], got32[-70:], *x.want(q[30:], [(0, range(1, 71))], 0.125))


@pytest.mark.parametrize("d,page", [(64, 32), (128, 128)])
def test_read_at_the_ends_of_32_bits(dev, d, page):
    """Positions outside the cache are NaN, the furthest an int32 names among them; rows that a sequence
    does not have stay as they were, and a row inside is still found."""
    x = Case(dev, 52, 2, d, page, [300, 300, 300, 300])
    k, _ = x.rows(300), x.rows(300)
    x.c.append(0, up(k, dev), up(k, dev), ints([0] * 4, dev), ints([0, 300, 300, 300, 300], dev))
    one = x.c.read(0, ints([299] * 4, dev), dtype=torch.float32)[0][0]
    assert torch.isfinite(one).all()
    for far in (2 ** 31 - 1, 2 ** 31 - 300, 2 ** 30, -2 ** 31, -2 ** 31 + 5, -2 ** 30, 1 << 20, -1 << 20):
        kk, vv = x.c.read(0, ints([299, far, far, far], dev), dtype=torch.float32)
        for y in (kk, vv):
            assert torch.equal(y[0], one) and torch.isnan(y[1:]).all(), far
        kk, vv = x.c.read(0, ints([299, far, far, -1], dev), ints([0, 1, 151, 401, 402], dev), total=405)
        for y in (kk, vv):
            assert torch.equal(y[0], one.to(torch.bfloat16)) and torch.isnan(y[1:402]).all(), far
    # the same positions are dropped by a write
    before = x.pool()
    for far in (2 ** 31 - 1, -2 ** 31, 2 ** 30, -2 ** 30):
        x.c.append(0, up(k, dev), up(k, dev), ints([far] * 4, dev), ints([0, 100, 150, 299, 300], dev))
        assert np.array_equal(x.pool(), before), far


def test_strides_of_single_rows_and_heads_say_nothing(dev):
    """K out of a fused projection's output and V alone: with one row, or one kv head, the strides that
    differ are never used."""
    x, y = (Case(dev, 53, 1, 64, 32, [40]) for _ in range(2))
    k, v = x.rows(1), x.rows(1)
    fused = torch.zeros((1, 3, 64), dtype=torch.bfloat16, device=dev)
    fused[:, 1:2] = up(k, dev)
    apart = up(v, dev).as_strided((1, 1, 64), (8, 8, 1))
    assert fused[:, 1:2].stride() != apart.stride()
    x.c.append(0, fused[:, 1:2], apart, ints([3], dev))
    y.c.append(0, up(k, dev), up(v, dev), ints([3], dev))
    assert np.array_equal(x.pool(), y.pool())
    dense = torch.zeros((1, 1, 40, 64), dtype=torch.bfloat16, device=dev)
    dense[0, 0, 9] = up(k, dev)[0, 0]
    wide = torch.zeros((1, 3, 40, 64), dtype=torch.bfloat16, device=dev)
    wide[0, 1, 9] = up(v, dev)[0, 0]
    x.c.append_cached(0, dense, wide[:, 1:2], ints([9], dev))
    y.c.append(0, up(k, dev), up(v, dev), ints([9], dev))
    assert np.array_equal(x.pool(), y.pool())
    z = Case(dev, 54, 2, 64, 32, [40])   # two kv heads: the head stride counts
    k = up(z.rows(2), dev)
    with pytest.raises(ValueError, match="layout"):
        z.c.append(0, k, k.transpose(0, 1).contiguous().transpose(0, 1), ints([0], dev), ints([0, 2], dev))
