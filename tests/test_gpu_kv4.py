"""The paged 4-bit K/V cache on the GPU against its numpy oracle: the pages' bytes exactly, what they
stand for exactly, attention within what fp32 through the codes allows, selected pages and page
bookkeeping exactly. Unwritten bytes of the pool are 0xFF throughout: scales that are NaN."""

import numpy as np
import pytest
import torch

from llmnputest_amd import kv4, ops
from oracle import kv4_oracle as ko

pytestmark = pytest.mark.gpu


def bf16(x):
    return ko.bf16_f32(ko.bf16_bits(np.asarray(x, np.float32)))


def up(x, dev):
    return torch.from_numpy(np.ascontiguousarray(x, np.float32)).to(dev).to(torch.bfloat16)


def ints(x, dev):
    return torch.tensor(list(x), dtype=torch.int32, device=dev)


def host(t):
    return t.float().cpu().numpy().astype(np.float64)


class Case:
    """A cache on the device, and its oracle, with pages dealt out in random order."""

    def __init__(self, dev, seed, hkv, d, page, need, spare=2, n_layers=1):
        self.rng = np.random.default_rng(seed)
        self.dev, self.hkv, self.d, self.page = dev, hkv, d, page
        cols = max(1, max(-(-n // page) for n in need))
        total = sum(-(-n // page) for n in need) + spare
        ids = self.rng.permutation(total)
        self.table = np.full((len(need), cols), -1, np.int32)
        at = 0
        for b, n in enumerate(need):
            k = -(-n // page)
            self.table[b, :k] = ids[at:at + k]
            at += k
        pool = torch.full((n_layers, total, kv4.page_bytes(page, hkv, d)), 255, dtype=torch.uint8, device=dev)
        refs = np.zeros(total, np.int32)
        refs[ids[:at]] = 1
        self.c = kv4.Kv4Cache.over(pool, torch.from_numpy(self.table).to(dev), ints([0] * len(need), dev),
                                   torch.from_numpy(refs).to(dev), n_kv_heads=hkv, head_dim=d, page_len=page)
        self.o = ko.Pages(pool[0].cpu().numpy().copy(), hkv, d, page)

    def rows(self, n, size=1.0):
        """Rows with channels of unlike size and offset."""
        a = np.exp(0.5 * self.rng.standard_normal((self.hkv, self.d)))
        z = 0.5 * self.rng.standard_normal((self.hkv, self.d))
        return bf16(size * (self.rng.standard_normal((n, self.hkv, self.d)) * a + z))

    def fill(self, lens, size=1.0):
        """Rows 0 .. lens[b] of every sequence, in both."""
        cu = np.concatenate([[0], np.cumsum(lens)])
        k, v = self.rows(max(1, cu[-1]), size), self.rows(max(1, cu[-1]), size)
        if cu[-1]:
            pos = [0] * len(lens)
            self.c.append(0, up(k, self.dev), up(v, self.dev), ints(pos, self.dev), ints(cu, self.dev))
            self.o.append(self.table, pos, [range(cu[i], cu[i + 1]) for i in range(len(lens))], k, v)
        return k, v

    def pool(self):
        return self.c.pool[0].cpu().numpy()

    def q(self, n, heads, size=1.0):
        return bf16(size * self.rng.standard_normal((n, heads, self.d)))

    def want(self, q, spans, scale, keep=None):
        """Oracle attention of the packed rows of q; spans[b] = (first row, end of each row)."""
        out, bound = np.zeros(q.shape), np.zeros(q.shape)
        for b, (at, ends) in enumerate(spans):
            n = len(ends)
            out[at:at + n], bound[at:at + n] = ko.attention(
                self.o, self.table[b], q[at:at + n].astype(np.float64), ends, scale,
                None if keep is None else keep[b])
        return out, bound


def check(got, got32, want, bound):
    """fp32 within the oracle's bound, bf16 within half a step more."""
    off = np.abs(host(got32) - want)
    assert (off <= bound + 1e-30).all(), (float((off - bound).max()), float(off.max()))
    off = np.abs(host(got) - want)
    assert (off <= bound + 2.0 ** -8 * (np.abs(want) + bound) + 1e-30).all()


# ------------------------------------------------------------------ rows

APPENDS = [  # hkv, d, page, [(first, then, then, ..) new rows of each sequence]
    (8, 64, 64, [(1,)]),
    (2, 64, 32, [(1, 1, 1), (31, 1, 1), (32, 1, 40)]),
    (3, 64, 64, [(5, 60, 70), (64, 64, 1), (0, 0, 3)]),
    (1, 64, 128, [(127, 1, 129), (128, 5, 0), (33, 31, 64)]),
    (2, 128, 64, [(63, 2, 1), (1, 62, 2)]),
    (1, 128, 32, [(15, 17, 1), (16, 16, 33), (7, 1, 100)]),
    (2, 128, 128, [(100, 29, 1)]),
]


@pytest.mark.parametrize("hkv,d,page,steps", APPENDS)
def test_append_bytes_and_read(dev, hkv, d, page, steps):
    """Ragged appends in several steps, each continuing inside a tile: the pool's bytes are the
    oracle's (those of no appended row too), and read() gives its values."""
    b = len(steps)
    x = Case(dev, 1, hkv, d, page, [sum(s) + 3 for s in steps])
    at = [0] * b
    for turn in range(len(steps[0])):
        new = [s[turn] for s in steps]
        cu = np.concatenate([[0], np.cumsum(new)])
        k, v = x.rows(cu[-1]), x.rows(cu[-1])
        x.c.append(0, up(k, dev), up(v, dev), ints(at, dev), ints(cu, dev), max_new=max(new))
        x.o.append(x.table, at, [range(cu[i], cu[i + 1]) for i in range(b)], k, v)
        assert np.array_equal(x.pool(), x.o.pool), turn
        for dt in (torch.float32, torch.bfloat16):
            kk, vv = x.c.read(0, ints(at, dev), ints(cu, dev), dtype=dt)
            for i in range(b):
                for j in range(new[i]):
                    p = at[i] + j
                    for h in range(hkv):
                        want = x.o.values(x.table[i, p // page], h, p % page)
                        for got, w in zip((kk, vv), want):
                            w = bf16(w) if dt == torch.bfloat16 else w
                            assert np.array_equal(got[cu[i] + j, h].float().cpu().numpy(), w)
        at = [a + n for a, n in zip(at, new)]


def test_append_one_row_each(dev):
    x = Case(dev, 2, 8, 64, 64, [200, 70, 1])
    for step, at in enumerate(([0, 0, 0], [1, 63, 0], [2, 64, 0], [199, 65, 0])):
        k, v = x.rows(3), x.rows(3)
        x.c.append(0, up(k, dev), up(v, dev), ints(at, dev))
        x.o.append(x.table, at, [[0], [1], [2]], k, v)
        assert np.array_equal(x.pool(), x.o.pool), step


def test_append_rewrites_and_rounds_as_written(dev):
    """A position written again takes the new row; values at the borders of a rounding; one group
    all alike; tiny and huge rows."""
    x = Case(dev, 3, 2, 64, 64, [128])
    for scale in (1.0, 1e-37, 3e36, 0.0):
        k = bf16(scale * np.round(x.rng.uniform(-8, 8, (100, 2, 64)) * 4) / 4)
        v = bf16(scale * np.arange(100 * 2 * 64).reshape(100, 2, 64) % 31)
        k[5] = v[7] = scale * 3
        k += 0.0   # no negative zeros: either is the least of zeros
        x.c.append(0, up(k, dev), up(v, dev), ints([0], dev), ints([0, 100], dev))
        x.o.append(x.table, [0], [range(100)], k, v)
        assert np.array_equal(x.pool(), x.o.pool), scale


def test_append_poison(dev):
    """NaN, infinities and a range past fp32: the group stands for NaN, its neighbours for themselves,
    and the page's bounds show it until the page begins again."""
    x = Case(dev, 4, 1, 64, 32, [64])
    k, v = x.rows(40), x.rows(40)
    k[3, 0, 5], k[4, 0, 40], v[6, 0, 63] = np.nan, np.inf, -np.inf
    k[34, 0, :2] = bf16([3e38, -3e38])
    x.c.append(0, up(k, dev), up(v, dev), ints([0], dev), ints([0, 40], dev))
    x.o.append(x.table, [0], [range(40)], k, v)
    assert np.array_equal(x.pool(), x.o.pool)
    kk, vv = x.c.read(0, ints([0], dev), ints([0, 40], dev), dtype=torch.float32)
    bad = torch.isnan(kk[:, 0]).cpu().numpy()
    want = np.zeros((40, 64), bool)
    want[3, :32] = want[4, 32:] = want[34, :32] = True
    assert np.array_equal(bad, want)
    want[:] = False
    want[6, 32:] = True
    assert np.array_equal(torch.isnan(vv[:, 0]).cpu().numpy(), want)
    assert np.isnan(ko.bf16_f32(x.o.bounds(x.table[0, 0], 0))).all()
    k = x.rows(1)
    x.c.append(0, up(k, dev), up(k, dev), ints([0], dev))
    x.o.append(x.table, [0], [[0]], k, k)
    assert np.array_equal(x.pool(), x.o.pool) and not np.isnan(ko.bf16_f32(x.o.bounds(x.table[0, 0], 0))).any()


def test_append_layouts(dev):
    """Strided rows (a fused projection's output), rows out of a dense cache at their positions, and a
    table of some of the sequences in another order."""
    x = Case(dev, 5, 2, 64, 64, [100, 130, 90])
    y = Case(dev, 5, 2, 64, 64, [100, 130, 90])
    assert np.array_equal(x.table, y.table)
    n = [90, 128, 77]
    cu = np.concatenate([[0], np.cumsum(n)])
    k, v = x.rows(cu[-1]), x.rows(cu[-1])
    both = torch.empty((cu[-1], 2, 2, 72), dtype=torch.bfloat16, device=dev)
    both[:, 0, :, :64], both[:, 1, :, :64] = up(k, dev), up(v, dev)
    x.c.append(0, both[:, 0, :, :64], both[:, 1, :, :64], ints([0] * 3, dev), ints(cu, dev))
    x.o.append(x.table, [0] * 3, [range(cu[i], cu[i + 1]) for i in range(3)], k, v)
    assert np.array_equal(x.pool(), x.o.pool)
    dk, dv = (torch.full((3, 2, 130, 64), float("nan"), dtype=torch.bfloat16, device=dev) for _ in range(2))
    for i in range(3):
        dk[i, :, :n[i]] = up(k[cu[i]:cu[i + 1]], dev).transpose(0, 1)
        dv[i, :, :n[i]] = up(v[cu[i]:cu[i + 1]], dev).transpose(0, 1)
    y.c.append_cached(0, dk, dv, ints([0] * 3, dev), ints(cu, dev))
    assert np.array_equal(y.pool(), x.o.pool)
    # one more row each, at its position, of sequences 2 and 0
    dk[0, :, 77] = dk[0, :, 3]
    dv[0, :, 77] = dv[0, :, 3]
    dk[1, :, 90] = dk[1, :, 4]
    dv[1, :, 90] = dv[1, :, 4]
    rows = y.c.table[[2, 0]].contiguous()
    y.c.append_cached(0, dk, dv, ints([77, 90], dev), table=rows)
    kk, vv = (torch.stack((t[0, :, 77], t[1, :, 90])).float().cpu().numpy() for t in (dk, dv))
    x.o.append(x.table[[2, 0]], [77, 90], [[0], [1]], kk, vv)
    assert np.array_equal(y.pool(), x.o.pool)


def test_append_outside_is_dropped(dev):
    """Positions the table does not hold, entries that name no page, rows the source does not have."""
    x = Case(dev, 6, 1, 64, 32, [64, 64])
    x.table[1, 0] = -1
    x.c.table[1, 0] = -1
    k, v = x.rows(20), x.rows(20)
    at = [58, 28]
    x.c.append(0, up(k, dev), up(v, dev), ints(at, dev), ints([0, 10, 20], dev))
    x.o.append(x.table, at, [range(10), range(10, 20)], k, v)
    assert np.array_equal(x.pool(), x.o.pool)
    x.c.append(0, up(k, dev), up(v, dev), ints([-3, 33], dev), ints([0, 4, 40], dev))   # 20 rows, not 40
    x.o.append(x.table, [-3, 33], [range(4), range(4, 20)], k, v)
    assert np.array_equal(x.pool(), x.o.pool)
    x.c.table[0, 1] = 1 << 20
    x.table[0, 1] = 1 << 20
    x.c.append(0, up(k, dev), up(v, dev), ints([40, 200], dev), ints([0, 9, 20], dev))
    assert np.array_equal(x.pool(), x.o.pool)
    kk, _ = x.c.read(0, ints([30, 62], dev), ints([0, 4, 8], dev))
    nan = torch.isnan(kk[:, 0, 0]).cpu().tolist()
    assert nan[2:4] == [True] * 2 and nan[6:] == [True] * 2   # no page; behind the table


# ------------------------------------------------------------------ attention, single tokens

DECODE = [  # hq, hkv, d, page, lens
    (40, 8, 64, 64, [513]),
    (5, 1, 64, 32, [1, 2, 31, 32, 33, 0, 64, 65]),
    (2, 2, 64, 64, [100, 63, 128]),
    (16, 1, 64, 128, [300, 1, 129]),
    (6, 2, 128, 32, [257, 40]),
    (8, 1, 128, 64, [1, 64, 191]),
    (3, 3, 128, 128, [500]),
    (4, 1, 64, 64, [1500]),
    (14, 2, 64, 64, [777, 3]),
]


@pytest.mark.parametrize("hq,hkv,d,page,lens", DECODE)
@pytest.mark.parametrize("n_split", [0, 1, 3])
def test_decode(dev, hq, hkv, d, page, lens, n_split):
    x = Case(dev, 7, hkv, d, page, [max(n, 1) for n in lens])
    x.fill(lens)
    q = x.q(len(lens), hq)
    got = x.c.attn(0, up(q, dev), ints(lens, dev), n_split=n_split, want_f32=True, scale=0.3)
    check(*got, *x.want(q, [(b, [n]) for b, n in enumerate(lens)], 0.3))
    for b, n in enumerate(lens):
        if n == 0:
            assert not got[1][b].any()


def test_decode_sharp_and_offset(dev):
    """Scores of hundreds, where one position has all the weight; keys with a large common offset."""
    x = Case(dev, 8, 2, 64, 64, [700])
    k, v = x.rows(700, 4.0) + 20, x.rows(700)
    k = bf16(k)
    x.c.append(0, up(k, dev), up(v, dev), ints([0], dev), ints([0, 700], dev))
    x.o.append(x.table, [0], [range(700)], k, v)
    q = x.q(1, 10, 3.0)
    check(*x.c.attn(0, up(q, dev), ints([700], dev), want_f32=True), *x.want(q, [(0, [700])], 0.125))


def test_decode_tiny_and_huge_values(dev):
    for size in (1e-30, 1e30):
        x = Case(dev, 9, 1, 64, 32, [99])
        k, v = x.rows(99), x.rows(99, size)
        x.c.append(0, up(k, dev), up(v, dev), ints([0], dev), ints([0, 99], dev))
        x.o.append(x.table, [0], [range(99)], k, v)
        q = x.q(1, 4)
        check(*x.c.attn(0, up(q, dev), ints([99], dev), want_f32=True), *x.want(q, [(0, [99])], 0.125))


def test_decode_shows_poison_and_missing_pages(dev):
    """A NaN in K that a token sees makes its heads NaN, one behind its length does not; a NaN in V its
    channels at least; an entry that names no page makes NaN; other sequences and kv heads are
    untouched."""
    x = Case(dev, 10, 2, 64, 32, [100, 100, 100, 100])
    k, v = x.rows(400), x.rows(400)
    k[50, 0, 3] = np.nan
    v[100 + 50, 1, 40] = np.inf
    cu = ints([0, 100, 200, 300, 400], dev)
    x.c.append(0, up(k, dev), up(v, dev), ints([0] * 4, dev), cu)
    x.c.table[3, 1] = -1
    q = up(x.q(4, 6), dev)
    out = x.c.attn(0, q, ints([100] * 4, dev))
    assert torch.isnan(out[0, :3]).all() and torch.isfinite(out[0, 3:]).all()
    assert torch.isnan(out[1, 3:, 32:]).all() and torch.isfinite(out[1, :3]).all()
    assert torch.isfinite(out[2]).all() and torch.isnan(out[3]).all()
    out = x.c.attn(0, q, ints([50, 50, 100, 32], dev))
    assert torch.isfinite(out).all()


def test_decode_lengths_beyond(dev):
    """lens past max_len reads max_len positions, past the table what the table holds; negative: none."""
    x = Case(dev, 11, 2, 64, 32, [96, 96, 96])
    x.fill([96, 96, 96])
    q = x.q(3, 4)
    got = x.c.attn(0, up(q, dev), ints([1000, 96, -5], dev), want_f32=True)
    check(*got, *x.want(q, [(0, [96]), (1, [96]), (2, [0])], 0.125))
    got = x.c.attn(0, up(q, dev), ints([1000, 50, 90], dev), max_len=70, want_f32=True)
    check(*got, *x.want(q, [(0, [70]), (1, [50]), (2, [70])], 0.125))


def test_decode_strided_queries_and_tables(dev):
    x = Case(dev, 12, 2, 64, 64, [200, 150, 90])
    x.fill([200, 150, 90])
    q = x.q(3, 6)
    wide = torch.zeros((3, 10, 64), dtype=torch.bfloat16, device=dev)
    wide[:, 2:8] = up(q, dev)
    lens = ints([200, 150, 90], dev)
    a = x.c.attn(0, up(q, dev), lens)
    assert torch.equal(x.c.attn(0, wide[:, 2:8], lens), a)
    order = torch.tensor([2, 0], device=dev)
    part = x.c.attn(0, up(q, dev)[order], lens[order], table=x.c.table[order], n_split=2)
    assert torch.equal(part, x.c.attn(0, up(q, dev), lens, n_split=2)[order])


def test_decode_no_sequence_depends_on_the_batch(dev):
    """Bit-identical runs, and a sequence's bits do not hang on its neighbours' lengths."""
    x = Case(dev, 13, 4, 64, 64, [900, 900])
    x.fill([900, 900])
    q = up(x.q(2, 20), dev)
    a = x.c.attn(0, q, ints([900, 700], dev), n_split=4)
    for _ in range(5):
        assert torch.equal(x.c.attn(0, q, ints([900, 700], dev), n_split=4), a)
    assert torch.equal(x.c.attn(0, q, ints([900, 3], dev), n_split=4)[0], a[0])


# ------------------------------------------------------------------ attention, blocks of tokens

PROMPT = [  # hq, hkv, d, page, [(tokens, length)]
    (5, 1, 64, 64, [(100, 100)]),
    (8, 2, 64, 32, [(33, 65), (1, 40), (0, 10), (2, 2)]),
    (4, 4, 64, 128, [(70, 300), (129, 129)]),
    (3, 1, 128, 32, [(40, 77), (65, 65)]),
    (16, 1, 64, 64, [(17, 200), (3, 3)]),
    (2, 1, 128, 128, [(200, 210)]),
    (1, 1, 64, 32, [(31, 31), (300, 333)]),
]


@pytest.mark.parametrize("hq,hkv,d,page,spans", PROMPT)
@pytest.mark.parametrize("n_split", [0, 2])
def test_prompt_blocks(dev, hq, hkv, d, page, spans, n_split):
    new, lens = zip(*spans)
    x = Case(dev, 20, hkv, d, page, lens)
    x.fill(lens)
    cu = np.concatenate([[0], np.cumsum(new)])
    q = x.q(cu[-1] + 3, hq)          # three rows behind the last sequence
    out = torch.full(q.shape, 7.0, dtype=torch.bfloat16, device=dev)
    got, got32 = x.c.attn(0, up(q, dev), ints(lens, dev), cu=ints(cu, dev), max_new=max(new), out=out,
                          n_split=n_split, want_f32=True)
    assert got is out and (got[cu[-1]:] == 7).all()
    want, bound = x.want(q, [(cu[b], [n - m + 1 + i for i in range(m)]) for b, (m, n) in enumerate(spans)],
                         d ** -0.5)
    check(got[:cu[-1]], got32[:cu[-1]], want[:cu[-1]], bound[:cu[-1]])


def test_prompt_rows_before_the_cache_are_zero(dev):
    """More tokens than positions: the first ones see nothing."""
    x = Case(dev, 21, 1, 64, 32, [40])
    x.fill([40])
    q = x.q(50, 2)
    got, got32 = x.c.attn(0, up(q, dev), ints([40], dev), cu=ints([0, 50], dev), want_f32=True)
    want, bound = x.want(q, [(0, [max(0, i - 9) for i in range(50)])], 0.125)
    check(got, got32, want, bound)
    assert not got[:10].any() and got[10].any()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n_split", [5, 17, 32, 63])
def test_blocks_merged_from_many_parts(dev, d, n_split):
    """Parts by the dozen (more than are weighed at a time among them), some of which some rows do not see
    at all, row blocks that end in the middle, and a sequence that is one part beside one of many."""
    x = Case(dev, 33, 1, d, 64, [2010, 40])
    x.fill([2010, 40])
    q, cu = x.q(53, 3, 3.0), [0, 50, 53]
    want, bound = x.want(q, [(0, range(1961, 2011)), (50, range(38, 41))], d ** -0.5)
    check(*x.c.attn(0, up(q, dev), ints([2010, 40], dev), cu=ints(cu, dev), n_split=n_split, want_f32=True),
          want, bound)
    q = x.q(2010, 3)
    rows = [0, 1, 31, 32, 500, 1279, 1999, 2009]
    got, got32 = x.c.attn(0, up(q, dev), ints([2010, 0], dev), cu=ints([0, 2010, 2010], dev), n_split=n_split,
                          want_f32=True)
    want, bound = ko.attention(x.o, x.table[0], q[rows].astype(np.float64), [r + 1 for r in rows], d ** -0.5)
    check(got[rows], got32[rows], want, bound)


def test_lengths_of_the_lowest_value(dev):
    """lens of -2^31: nothing is seen, by single tokens and by blocks."""
    x = Case(dev, 27, 2, 64, 32, [40, 40])
    x.fill([40, 40])
    low = ints([-2 ** 31, 40], dev)
    out = x.c.attn(0, up(x.q(2, 4), dev), low)
    assert not out[0].any() and out[1].any()
    for n_split in (0, 2):
        out = x.c.attn(0, up(x.q(300, 4), dev), low, cu=ints([0, 260, 300], dev), n_split=n_split)
        assert not out[:260].any() and out[260:].any()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("scale", [0.0, -0.7])
def test_scales_of_any_sign(dev, d, scale):
    x = Case(dev, 28, 1, d, 64, [130, 33])
    x.fill([130, 33])
    q = x.q(2, 5)
    got = x.c.attn(0, up(q, dev), ints([130, 33], dev), scale=scale, want_f32=True)
    check(*got, *x.want(q, [(0, [130]), (1, [33])], scale))
    q = x.q(60, 5)
    got = x.c.attn(0, up(q, dev), ints([130, 33], dev), cu=ints([0, 50, 60], dev), scale=scale, want_f32=True)
    check(*got, *x.want(q, [(0, range(81, 131)), (50, range(24, 34))], scale))


@pytest.mark.parametrize("n_seqs,d", [(65, 64), (700, 128), (2100, 64)])
def test_many_sequences(dev, n_seqs, d):
    """More sequences than a wave has lanes, and (2100 x 8 kv heads) more than there are counters."""
    hkv = 8 if n_seqs == 2100 else 1
    lens = np.random.default_rng(3).integers(0, 70, n_seqs)
    lens[:3] = [0, 69, 64]
    x = Case(dev, 29, hkv, d, 32, lens)
    some = [0, 1, 2, 62, 63, 64] + ([127, 128, n_seqs - 2, n_seqs - 1] if n_seqs > 65 else [])
    at = np.concatenate([[0], np.cumsum(lens)])
    k, v = x.rows(at[-1]), x.rows(at[-1])
    x.c.append(0, up(k, dev), up(v, dev), ints([0] * n_seqs, dev), ints(at, dev), max_new=69)
    x.o.append(x.table[some], [0] * len(some), [range(at[b], at[b + 1]) for b in some], k, v)
    q = x.q(n_seqs, 2 * hkv)
    got = x.c.attn(0, up(q, dev), ints(lens, dev), want_f32=True)
    new = np.minimum(lens, np.random.default_rng(4).integers(0, 6, n_seqs))
    cu = np.concatenate([[0], np.cumsum(new)])
    qb = x.q(cu[-1], 2 * hkv)
    block = x.c.attn(0, up(qb, dev), ints(lens, dev), cu=ints(cu, dev), max_new=5, want_f32=True)
    for b in some:
        want, bound = ko.attention(x.o, x.table[b], q[b:b + 1].astype(np.float64), [int(lens[b])], d ** -0.5)
        check(got[0][b:b + 1], got[1][b:b + 1], want, bound)
        if new[b]:
            rows = slice(cu[b], cu[b + 1])
            want, bound = ko.attention(x.o, x.table[b], qb[rows].astype(np.float64),
                                       range(int(lens[b] - new[b]) + 1, int(lens[b]) + 1), d ** -0.5)
            check(block[0][rows], block[1][rows], want, bound)


@pytest.mark.parametrize("n_seqs,tiles,d", [(1024, 8, 64), (1100, 2, 128), (120, 20, 64), (100, 35, 64),
                                            (80, 260, 64), (70, 70, 128)])
def test_many_short_sequences_share_a_line(dev, n_seqs, tiles, d):
    """More than 16384 tiles in (sequence, kv head)s of at most eight: some end one workgroup's stretch and
    begin the next. All sequences name the same pages and ask the same, so that those of one length are
    alike."""
    x = Case(dev, 32, 8, d, 32, [32 * tiles], spare=0)
    x.fill([32 * tiles])
    lens = np.random.default_rng(6).integers(32 * tiles - 40, 32 * tiles + 1, n_seqs)
    table = x.c.table.expand(n_seqs, tiles).contiguous()
    q = np.repeat(x.q(1, 8), n_seqs, 0)
    out, out32 = x.c.attn(0, up(q, dev), ints(lens, dev), table=table, want_f32=True)
    for n in np.unique(lens)[::13]:
        want, bound = ko.attention(x.o, x.table[0], q[:1].astype(np.float64), [int(n)], d ** -0.5)
        rows = torch.from_numpy(np.flatnonzero(lens == n)).to(dev)
        check(out[rows], out32[rows], want, bound)


def test_more_tiles_than_workgroups_times_words(dev):
    """2048 sequences x 8 kv heads over 2^18 positions each, all of them one page again and again: the
    launch has more workgroups than share the line of tiles, and a workgroup's place times its share
    passes 2^31. What is seen is the page's 128 positions, 2048 times each: the page's own attention. The
    bound grows with the tiles summed, 8192 + 80 of them for the oracle's 4 + 80."""
    x = Case(dev, 30, 8, 64, 128, [128], spare=0)
    x.fill([128])
    n, pages = 2048, 2048
    c = kv4.Kv4Cache.over(x.c.pool, torch.zeros((n, pages), dtype=torch.int32, device=dev),
                          ints([pages * 128] * n, dev), x.c.refs, n_kv_heads=8, head_dim=64, page_len=128)
    q = x.q(n, 8)
    out, out32 = c.attn(0, up(q, dev), want_f32=True)
    for b in (0, 1, 700, 1023, 1024, n - 1):
        want, bound = ko.attention(x.o, x.table[0], q[b:b + 1].astype(np.float64), [128], 0.125)
        check(out[b:b + 1], out32[b:b + 1], want, bound * (8272 / 84))
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("d,n_split", [(64, 0), (64, 3), (128, 0)])
def test_blocks_are_the_same_every_time(dev, d, n_split):
    """Neither the order in which workgroups end nor what runs beside them changes a bit."""
    x = Case(dev, 31, 2, d, 64, [700, 1500])
    x.fill([700, 1500])
    cu, lens, q = ints([0, 300, 1000], dev), ints([700, 1500], dev), up(x.q(1000, 10), dev)
    one = up(x.q(2, 10), dev)
    first, token = x.c.attn(0, q, lens, cu=cu, n_split=n_split), x.c.attn(0, one, lens)
    for _ in range(30):
        assert torch.equal(x.c.attn(0, q, lens, cu=cu, n_split=n_split), first)
        assert torch.equal(x.c.attn(0, one, lens), token)


def test_prompt_poison_is_causal(dev):
    """A NaN at a position shows in the tokens that see it, not in those before it."""
    x = Case(dev, 22, 1, 64, 32, [90, 90])
    k, v = x.rows(180), x.rows(180)
    k[70, 0, 0] = np.nan
    v[90 + 33, 0, 2] = np.nan
    x.c.append(0, up(k, dev), up(v, dev), ints([0, 0], dev), ints([0, 90, 180], dev))
    out = x.c.attn(0, up(x.q(180, 4), dev), ints([90, 90], dev), cu=ints([0, 90, 180], dev), max_new=90)
    assert torch.isfinite(out[:70]).all() and torch.isnan(out[70:90]).all()
    assert torch.isfinite(out[90:123]).all() and torch.isnan(out[123:, :, :32]).all()


def test_prompt_equals_its_tokens(dev):
    """A block's rows and the same tokens one at a time agree within both bounds."""
    x = Case(dev, 23, 2, 64, 64, [150])
    x.fill([150])
    q = x.q(20, 8)
    _, a = x.c.attn(0, up(q, dev), ints([150], dev), cu=ints([0, 20], dev), want_f32=True)
    want, bound = x.want(q, [(0, [131 + i for i in range(20)])], 0.125)
    for i in range(20):
        _, b = x.c.attn(0, up(q[i:i + 1], dev), ints([131 + i], dev), want_f32=True)
        assert (np.abs(host(b[0]) - host(a[i])) <= 2 * bound[i]).all()


# ------------------------------------------------------------------ selected pages

SELECT = [  # hq, hkv, d, page, lens, n_sel, first, last
    (5, 1, 64, 32, [500, 33, 1, 0, 96], 6, 1, 1),
    (8, 2, 64, 64, [1000, 64], 4, 0, 0),
    (6, 2, 128, 32, [700], 9, 2, 3),
    (16, 1, 128, 64, [640, 300], 3, 1, 2),
    (4, 4, 64, 128, [1400], 200, 1, 1),
    (2, 1, 64, 32, [4000], 100, 0, 1),
]


@pytest.mark.parametrize("hq,hkv,d,page,lens,n_sel,first,last", SELECT)
def test_select_and_attention(dev, hq, hkv, d, page, lens, n_sel, first, last):
    x = Case(dev, 30, hkv, d, page, [max(n, 1) for n in lens])
    x.fill(lens)
    q = x.q(len(lens), hq)
    sel = x.c.select(0, up(q, dev), ints(lens, dev), n_sel, first, last)
    want = np.stack([ko.select(x.o, x.table[b], q[b].astype(np.float64), n, n_sel, first, last)
                     for b, n in enumerate(lens)])
    assert np.array_equal(sel.cpu().numpy(), want)
    for ns in (0, 3):
        got = x.c.attn(0, up(q, dev), ints(lens, dev), sel=sel, n_split=ns, want_f32=True)
        keep = [[set(w[w >= 0].tolist()) for w in want[b]] for b in range(len(lens))]
        check(*got, *x.want(q, [(b, [n]) for b, n in enumerate(lens)], d ** -0.5, keep))


def test_select_ties_and_zero_queries(dev):
    """Pages alike in every bound, scores of +0 and -0: the lowest pages first."""
    x = Case(dev, 31, 2, 64, 32, [32 * 20])
    k = np.tile(x.rows(32), (20, 1, 1))
    x.c.append(0, up(k, dev), up(k, dev), ints([0], dev), ints([0, 640], dev))
    x.o.append(x.table, [0], [range(640)], k, k)
    for q in (x.q(1, 4), np.zeros((1, 4, 64), np.float32), np.full((1, 4, 64), -0.0, np.float32)):
        sel = x.c.select(0, up(q, dev), ints([640], dev), 7, 0, 1).cpu().numpy()
        assert (sel == [0, 1, 2, 3, 4, 5, 19]).all()


def test_select_poison_comes_after_the_pages_always_read(dev):
    x = Case(dev, 32, 1, 64, 32, [320])
    k, v = x.rows(320), x.rows(320)
    k[32 * 6 + 3, 0, 9] = np.nan
    x.c.append(0, up(k, dev), up(v, dev), ints([0], dev), ints([0, 320], dev))
    q = up(x.q(1, 3), dev)
    assert x.c.select(0, q, ints([320], dev), 3, 1, 1).cpu().tolist() == [[[0, 6, 9]]]
    assert x.c.select(0, q, ints([320], dev), 2, 1, 1).cpu().tolist() == [[[0, 9]]]
    q[0, 0, 0] = float("nan")     # every page's score: the lowest of them
    assert x.c.select(0, q, ints([320], dev), 4, 1, 1).cpu().tolist() == [[[0, 1, 2, 9]]]


def test_select_as_many_pages_as_it_takes(dev):
    """16384 pages in one row of the table (pages repeat: ties everywhere but at their bounds)."""
    x = Case(dev, 33, 1, 64, 32, [32 * 50])
    x.fill([32 * 50])
    ids = x.rng.integers(0, 50, 16384)
    big = torch.from_numpy(x.table[0, ids][None].copy()).to(dev)
    q = x.q(1, 2)
    n = 16384 * 32 - 5
    sel = x.c.select(0, up(q, dev), ints([n], dev), 700, 1, 1, table=big).cpu().numpy()[0]
    assert np.array_equal(sel, ko.select(x.o, x.table[0, ids], q[0].astype(np.float64), n, 700, 1, 1))


def test_sel_of_the_callers_own(dev):
    """Lists in any order, with entries that are none, outside the sequence, or all of them."""
    x = Case(dev, 34, 2, 64, 32, [150, 100])
    x.fill([150, 100])
    q = x.q(2, 6)
    sel = torch.tensor([[[4, -1, 0, 9, 2], [-1, -1, -1, -1, -1]], [[3, 2, 1, 0, 4], [1 << 30, 7, -9, 1, 5]]],
                       dtype=torch.int32, device=dev)
    keep = [[{4, 0, 2}, set()], [{0, 1, 2, 3}, {1}]]
    got = x.c.attn(0, up(q, dev), ints([150, 100], dev), sel=sel, want_f32=True)
    check(*got, *x.want(q, [(0, [150]), (1, [100])], 0.125, keep))
    assert not got[0][0, 3:].any()


# ------------------------------------------------------------------ pages

def same(c, book):
    assert np.array_equal(c.table.cpu().numpy(), book.table)
    assert np.array_equal(c.lens.cpu().numpy(), book.lens)
    assert np.array_equal(c.refs.cpu().numpy(), book.refs)


@pytest.mark.parametrize("seed,n_seqs,n_pages,page,layers", [(0, 6, 40, 32, 3), (1, 20, 60, 64, 1),
                                                             (2, 3, 9, 32, 2), (3, 12, 5000, 32, 1),
                                                             (4, 30, 13, 128, 1)])
def test_bookkeeping(dev, seed, n_seqs, n_pages, page, layers):
    """A long random run of reserve, fork, free and compact: tables, counts, statuses and every byte of
    the pool as the oracle's."""
    rng = np.random.default_rng(seed)
    cols = 12
    c = kv4.Kv4Cache(layers, n_pages, n_seqs, cols * page, n_kv_heads=1, page_len=page, device=dev)
    c.pool.copy_(torch.randint(0, 256, c.pool.shape, dtype=torch.uint8, device=dev))
    pool, book = c.pool.cpu().numpy().copy(), ko.Book(n_seqs, cols, n_pages, page)
    for turn in range(40):
        what = turn if turn < 2 else rng.integers(0, 5)
        if what <= 1:
            want = rng.integers(-3, (cols + 1) * page, n_seqs) * (rng.random(n_seqs) < 0.4)
            c.reserve(want.tolist())
            bad = book.reserve(want)
            have = (book.table >= 0).sum(1) * page
            book.lens[:] = np.minimum(np.maximum(book.lens, want), have)
            c.lens.copy_(torch.from_numpy(book.lens))
        elif what == 2:
            n = int(rng.integers(1, min(n_seqs, 6) + 1))
            src, dst = rng.integers(-1, n_seqs + 1, n).tolist(), rng.integers(-1, n_seqs + 1, n).tolist()
            c.fork(src, dst)
            bad = book.fork(src, dst)
        elif what == 3:
            seqs = rng.integers(-1, n_seqs + 1, int(rng.integers(1, 4))).tolist()
            c.free(seqs)
            bad = book.free(seqs)
        else:
            live = c.compact()
            bad = int(c.status)
            assert int(live) == book.compact()
        for a, z in book.moves:
            pool[:, z] = pool[:, a]
        book.moves.clear()
        same(c, book)
        assert int(c.status) == bad, (turn, what)
        assert np.array_equal(c.pool.cpu().numpy(), pool), (turn, what)


def test_copy_pages(dev):
    c = kv4.Kv4Cache(3, 20, 1, 64, n_kv_heads=3, head_dim=128, page_len=32, device=dev)
    c.pool.copy_(torch.randint(0, 256, c.pool.shape, dtype=torch.uint8, device=dev))
    want = c.pool.clone()
    want[:, [5, 6, 7]] = want[:, [0, 19, 0]]
    c.copy_pages([0, 19, 0, -1, 3, 20, 8], [5, 6, 7, 2, 20, 1, 8])
    assert torch.equal(c.pool, want)


def test_pool_with_layers_inside_pages(dev):
    """A pool laid out [pages][layers]: the layer stride is smaller than the pages'."""
    size = kv4.page_bytes(32, 1, 64)
    mem = torch.randint(0, 256, (10, 4, size), dtype=torch.uint8, device=dev)
    c = kv4.Kv4Cache.over(mem.transpose(0, 1), torch.full((3, 4), -1, dtype=torch.int32, device=dev),
                          ints([0] * 3, dev), ints([0] * 10, dev), n_kv_heads=1, page_len=32)
    c.reserve([40, 0, 33])
    c.lens.copy_(ints([40, 0, 33], dev))
    want = mem.clone()
    c.fork([0], [1])
    want[4] = want[1]
    assert torch.equal(mem, want) and c.table[:, :2].cpu().tolist() == [[0, 1], [0, 4], [2, 3]]
    c.free([0])
    assert int(c.compact()) == 4
    want[1] = want[4]
    assert torch.equal(mem, want) and c.table[:, :2].cpu().tolist() == [[-1, -1], [0, 1], [2, 3]]


# ------------------------------------------------------------------ together, streams, graphs

def test_serving_run(dev):
    """Prompts, steps, a fork that goes its own way, sequences that end, a compaction: attention agrees
    with the oracle at every point, and moving pages changes no bit of it."""
    page, hkv, hq = 32, 2, 8
    x = Case(dev, 40, hkv, 64, page, [1], spare=0)
    c = kv4.Kv4Cache(2, 40, 4, 6 * page, n_kv_heads=hkv, page_len=page, device=dev)
    c.pool.fill_(255)
    o = ko.Pages(c.pool[1].cpu().numpy().copy(), hkv, 64, page)
    book = ko.Book(4, 6, 40, page)
    x.o = o

    def sync():
        for a, z in book.moves:
            o.pool[z] = o.pool[a]
        book.moves.clear()
        same(c, book)
        x.table = book.table

    def put(pos, new):
        cu = np.concatenate([[0], np.cumsum(new)])
        k, v = x.rows(cu[-1]), x.rows(cu[-1])
        c.append(1, up(k, dev), up(v, dev), ints(pos, dev), ints(cu, dev), max_new=max(new))
        o.append(book.table, pos, [range(cu[i], cu[i + 1]) for i in range(4)], k, v)
        book.lens[:] = [p + n for p, n in zip(pos, new)]
        c.lens.copy_(torch.from_numpy(book.lens))
        q = x.q(cu[-1], hq)
        got = c.attn(1, up(q, dev), cu=ints(cu, dev), max_new=max(new), want_f32=True)
        spans = [(cu[b], [pos[b] + 1 + i for i in range(new[b])]) for b in range(4)]
        check(*got, *x.want(q, spans, 0.125))

    c.reserve([100, 60, 0, 0])
    book.reserve([100, 60, 0, 0])
    sync()
    put([0, 0, 0, 0], [77, 50, 0, 0])
    c.fork([0, 1], [2, 3])
    book.fork([0, 1], [2, 3])
    sync()
    c.reserve([120, 80, 110, 90])
    book.reserve([120, 80, 110, 90])
    sync()
    for step in range(3):
        put(book.lens.tolist(), [1, 1, 1, 1])
    put(book.lens.tolist(), [20, 0, 13, 1])
    c.free([0, 3])
    book.free([0, 3])
    sync()
    q = up(x.q(4, hq), dev)
    before = c.attn(1, q)
    sel = c.select(1, q, n_sel=3)
    sparse = c.attn(1, q, sel=sel)
    live = c.compact()
    assert int(live) == book.compact()
    sync()
    assert torch.equal(c.attn(1, q), before) and not before[0].any() and not before[3].any()
    assert torch.equal(c.select(1, q, n_sel=3), sel) and torch.equal(c.attn(1, q, sel=sel), sparse)
    assert np.array_equal(c.pool[1].cpu().numpy()[:int(live)], o.pool[:int(live)])
    put(book.lens.tolist(), [0, 5, 2, 0])


def test_graph_replays_and_eager_calls(dev):
    """append, select, both attentions, and the bookkeeping of a step captured in a graph, replayed
    among eager calls that use the default workspace: every replay equals the eager result."""
    x = Case(dev, 41, 2, 64, 32, [1000, 600])
    x.fill([900, 500])
    q, k, v = up(x.q(2, 10), dev), up(x.rows(2), dev), up(x.rows(2), dev)
    pos, lens = ints([900, 500], dev), ints([901, 501], dev)
    cu = ints([0, 20, 33], dev)
    block = up(x.q(33, 10), dev)

    def step():
        x.c.append(0, k, v, pos)
        sel = x.c.select(0, q, lens, n_sel=7)
        return (sel, x.c.attn(0, q, lens, n_split=5), x.c.attn(0, q, lens, sel=sel, n_split=3),
                x.c.attn(0, block, lens, cu=cu, max_new=20), *x.c.read(0, pos))

    want = [t.clone() for t in step()]
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    side = torch.cuda.Stream()
    for rep in range(5):
        for t in got:
            t.zero_()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            g.replay()
        eager = step()
        torch.cuda.synchronize()
        for a, b, w in zip(got, eager, want):
            assert torch.equal(a, w) and torch.equal(b, w), rep
        pos.add_(0)


def test_page_ops_in_a_graph(dev):
    c = kv4.Kv4Cache(2, 30, 4, 320, n_kv_heads=1, page_len=32, device=dev)
    c.pool.copy_(torch.randint(0, 256, c.pool.shape, dtype=torch.uint8, device=dev))
    c.reserve([100, 70, 0, 0])
    c.lens.copy_(ints([100, 70, 0, 0], dev))
    keep = [t.clone() for t in (c.pool, c.table, c.lens, c.refs)]
    src, dst, gone, want = ints([0, 1], dev), ints([2, 3], dev), ints([0], dev), ints([0, 80, 130, 80], dev)

    def step():
        for t, s in zip((c.pool, c.table, c.lens, c.refs), keep):
            t.copy_(s)
        c.fork(src, dst)
        c.reserve(want)
        c.free(gone)
        return c.compact()

    live = int(step())
    after = [t.clone() for t in (c.pool, c.table, c.lens, c.refs)]
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for rep in range(4):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert int(out) == live
        for t, s in zip((c.pool, c.table, c.lens, c.refs), after):
            assert torch.equal(t, s), rep
        assert int(step()) == live


def test_streams_at_once(dev):
    """Calls without a workspace of their own on several streams: the bits of the same calls alone."""
    x = Case(dev, 42, 4, 64, 64, [1200, 1200, 1200])
    x.fill([1200, 1000, 800])
    lens = ints([1200, 1000, 800], dev)
    qs = [up(x.q(3, 20), dev) for _ in range(4)]
    want = [(x.c.attn(0, q, lens, n_split=6), x.c.select(0, q, lens, n_sel=5)) for q in qs]
    streams = [torch.cuda.Stream() for _ in qs]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[] for _ in qs]
    for _ in range(10):
        for s, q, g in zip(streams, qs, got):
            with torch.cuda.stream(s):
                g.append((x.c.attn(0, q, lens, n_split=6), x.c.select(0, q, lens, n_sel=5)))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        for pair in g:
            assert torch.equal(pair[0], w[0]) and torch.equal(pair[1], w[1])


def test_pages_past_32_bits(dev):
    """A pool whose last pages lie more than 4 GiB behind its first."""
    size = kv4.page_bytes(128, 8, 128)
    n = (1 << 32) // size + 40
    pool = torch.empty((1, n, size), dtype=torch.uint8, device=dev)
    c = kv4.Kv4Cache.over(pool, torch.tensor([[n - 1, 0, n - 2], [1, n - 3, 2]], dtype=torch.int32, device=dev),
                          ints([0, 0], dev), torch.zeros(n, dtype=torch.int32, device=dev), n_kv_heads=8,
                          head_dim=128, page_len=128)
    small = kv4.Kv4Cache(1, 6, 2, 384, n_kv_heads=8, head_dim=128, page_len=128, device=dev)
    small.table.copy_(torch.tensor([[0, 1, 2], [3, 4, 5]], dtype=torch.int32))
    x = Case(dev, 43, 8, 128, 128, [1])
    k, v = up(x.rows(700), dev), up(x.rows(700), dev)
    q = up(x.q(2, 16), dev)
    lens = ints([380, 320], dev)
    outs = []
    for cache in (c, small):
        cache.append(0, k, v, ints([0, 0], dev), ints([0, 380, 700], dev))
        outs.append((cache.attn(0, q, lens), cache.select(0, q, lens, n_sel=2),
                     *cache.read(0, ints([0, 0], dev), ints([0, 380, 700], dev))))
    for a, b in zip(*outs):
        assert torch.equal(a, b)
    c.copy_pages([n - 1], [7])
    assert torch.equal(pool[0, 7], pool[0, n - 1])


# ------------------------------------------------------------------ refusals

def test_python_refusals(dev):
    c = kv4.Kv4Cache(2, 8, 2, 128, n_kv_heads=2, page_len=32, device=dev)
    z = lambda *s, dt=torch.bfloat16: torch.zeros(s, dtype=dt, device=dev)   # noqa: E731
    k, q, one = z(2, 2, 64), z(2, 4, 64), ints([0, 0], dev)
    with pytest.raises(IndexError):
        c.append(2, k, k, one)
    for bad in (z(2, 3, 64), z(2, 2, 32), z(2, 2, 128)[:, :, ::2]):
        with pytest.raises(ValueError):
            c.append(0, bad, bad, one)
    with pytest.raises(TypeError):
        c.append(0, k.float(), k.float(), one)
    with pytest.raises(ValueError, match="layout"):
        c.append(0, k, z(3, 2, 64), one)
    with pytest.raises(ValueError, match="sequences"):
        c.append(0, z(3, 2, 64), z(3, 2, 64), one)
    with pytest.raises(ValueError):
        c.append(0, k, k, ints([0], dev))
    with pytest.raises(TypeError):
        c.append(0, k, k, one.long())
    with pytest.raises(ValueError):
        c.append(0, k, k, one.cpu())
    with pytest.raises(ValueError):
        c.append(0, k, k, one, cu=ints([0, 1], dev))
    with pytest.raises(ops._lib.Q4NXError):        # rows that are not 16 bytes apart
        c.append(0, z(2, 2, 66)[:, :, :64], z(2, 2, 66)[:, :, :64], one)
    with pytest.raises(ValueError):
        c.append_cached(0, z(1, 2, 9, 64), z(1, 2, 9, 64), one)
    with pytest.raises(TypeError):
        c.read(0, one, dtype=torch.float16)
    for bad in (z(2, 4, 32), z(4, 64), z(2, 8, 64)[:, ::2], z(3, 4, 64)):
        with pytest.raises(ValueError):
            c.attn(0, bad, one)
    with pytest.raises(ops._lib.Q4NXError):
        c.attn(0, z(2, 5, 64), one)
    with pytest.raises(ops._lib.Q4NXError):
        c.attn(0, z(2, 34, 64), one)               # 17 heads per kv head
    with pytest.raises(ValueError, match="sel"):
        c.attn(0, q, one, sel=z(2, 3, 4, dt=torch.int32))
    with pytest.raises(ops._lib.Q4NXError):        # a page list for a block of tokens
        c.attn(0, q, one, cu=ints([0, 2, 2], dev), max_new=2, sel=z(2, 2, 4, dt=torch.int32))
    with pytest.raises(ValueError, match="out"):
        c.attn(0, q, one, out=z(2, 4, 128)[:, :, :64])
    with pytest.raises(ops._lib.Q4NXError):
        c.select(0, q, one, n_sel=1)               # does not hold the first and the last page
    with pytest.raises(ValueError):
        c.select(0, z(3, 4, 64), one)
    with pytest.raises(ValueError):
        c.fork([0], [1, 1])
    with pytest.raises(ValueError):
        c.reserve([1])
    with pytest.raises(ValueError):
        c.free([0, 1, 1])
    with pytest.raises(ValueError):
        kv4.Kv4Cache.over(c.pool, c.table, c.lens[:1], c.refs, n_kv_heads=2, page_len=32)
    with pytest.raises(ValueError):
        kv4.Kv4Cache.over(c.pool, c.table, c.lens, c.refs, n_kv_heads=1, page_len=32)
    c.append(0, z(0, 2, 64), z(0, 2, 64), one, cu=ints([0, 0, 0], dev))   # nothing to do
    assert c.attn(0, z(0, 4, 64), one, cu=ints([0, 0, 0], dev)).shape == (0, 4, 64)


def test_a_row_shown_twice_is_refused(dev):
    c = kv4.Kv4Cache(1, 8, 2, 128, n_kv_heads=2, page_len=32, device=dev)
    twice = c.table[:1].expand(2, 4)
    one, q = ints([0, 0], dev), torch.zeros((2, 4, 64), dtype=torch.bfloat16, device=dev)
    for f in (lambda: c.attn(0, q, one, table=twice), lambda: c.select(0, q, one, n_sel=2, table=twice),
              lambda: c.append(0, q[:, :2], q[:, :2], one, table=twice), lambda: c.read(0, one, table=twice)):
        with pytest.raises(ops._lib.Q4NXError, match="stride"):
            f()
    with pytest.raises(ops._lib.Q4NXError, match="stride"):
        kv4.Kv4Cache.over(c.pool, twice, c.lens, c.refs, n_kv_heads=2, page_len=32).read(0, one)
