"""Single tokens of many sequences of clearly unequal lengths, shared out by the lengths as the kernel
finds them (no n_split): in parts and on one line, with fewer and more sequences than a wave has lanes.
A few pages stand behind every sequence, again and again, so that contexts are long and the oracle small:
what a sequence sees is each cached position a number of times."""

import numpy as np
import pytest
import torch

from tests.test_gpu_kv4 import Case, check, ints, up

pytestmark = pytest.mark.gpu

PAGES = 3


class Round:
    """Sequences of PAGES pages, repeated; one softmax over the positions with their counts."""

    def __init__(self, dev, seed, hkv, group, d, page, n_seqs, longest):
        self.x = Case(dev, seed, hkv, d, page, [PAGES * page], spare=1)
        self.x.fill([PAGES * page])
        self.hkv, self.group, self.d, self.span = hkv, group, d, PAGES * page
        cols = -(-longest // page)
        row = self.x.c.table[0, torch.arange(cols, device=dev) % PAGES]
        self.table = row.expand(n_seqs, cols).contiguous()
        at, table, o = range(self.span), self.x.table[0], self.x.o
        kv = [[o.values(table[p // page], h, p % page) for p in at] for h in range(hkv)]
        sc = [[o.scales(table[p // page], h, p % page) for p in at] for h in range(hkv)]
        self.k, self.v = (np.array([[y[i] for y in r] for r in kv], np.float64) for i in (0, 1))
        # [hkv, positions, d]: steps and offsets of K, then of V
        self.dk, self.dv = (np.repeat([[y[0][i] for y in r] for r in sc], 32, -1) for i in (0, 1))
        self.mk, self.mv = (np.repeat([[y[1][i] for y in r] for r in sc], 32, -1) for i in (0, 1))

    def want(self, q, n, scale):
        """One sequence of n positions, q [heads, d]: (out, bound). The bound's terms are those of the
        oracle's attention (scores through 128 + code, p d in two bf16 terms, sums over the tiles, at most 80
        more in the merge)."""
        out, bound = np.zeros(q.shape), np.zeros(q.shape)
        count = n // self.span + (np.arange(self.span) < n % self.span)
        see = count > 0
        tiles = -(-n // 32) + 80
        for i in range(len(q)) if n else ():
            h = i // self.group
            k, v, dk, mk, dv, mv = (y[h][see] for y in (self.k, self.v, self.dk, self.mk, self.dv, self.mv))
            s = scale * (k @ q[i])
            p = count[see] * np.exp(s - s.max())
            p /= p.sum()
            out[i] = p @ v
            es = (abs(scale) * ((143 * dk + mk) @ np.abs(q[i])) * 40 + 4 * np.abs(s)) * 2.0 ** -24
            bound[i] = (2 * es.max() + 2.0 ** -20 + tiles * 2.0 ** -24) * (p @ (15 * dv + mv)) \
                + (p @ dv) * 31 * (2.0 ** -18 + tiles * 2.0 ** -24) + (p @ mv) * tiles * 2.0 ** -24
        return out, bound

    def run(self, lens, repeat=2):
        """The kernel's rows of every sequence against the oracle's, and the same bits again."""
        dev, scale = self.x.dev, self.d ** -0.5
        q = self.x.q(len(lens), self.hkv * self.group)
        got = self.x.c.attn(0, up(q, dev), ints(lens, dev), table=self.table, want_f32=True)
        for _ in range(repeat):
            assert torch.equal(self.x.c.attn(0, up(q, dev), ints(lens, dev), table=self.table), got[0])
        want, bound = (np.stack(y) for y in zip(*(self.want(q[b].astype(np.float64), int(n), scale)
                                                  for b, n in enumerate(lens))))
        check(*got, want, bound)
        empty = np.asarray(lens) == 0
        assert not got[1][torch.from_numpy(empty).to(dev)].any()


PARTS = [  # hkv, group, d, page, lens: a longest one of more than 32 tiles, too few tiles for a line
    (2, 5, 64, 64, [3000, 0, 1, 33, 2047, 500, 1025, 2999]),
    (1, 3, 128, 32, [2999, 31, 0, 32, 1500, 3000, 64, 2]),
    (4, 16, 64, 128, [1, 0, 2900, 0, 0, 3001, 7, 129]),
    (8, 4, 128, 64, [9000, 20, 0, 1]),
    (1, 1, 64, 32, [0, 1025, 0]),
]


@pytest.mark.parametrize("hkv,group,d,page,lens", PARTS)
def test_few_ragged_sequences_in_parts(dev, hkv, group, d, page, lens):
    r = Round(dev, 60, hkv, group, d, page, len(lens), max(lens))
    r.run(lens)
    r.run(lens[::-1])


@pytest.mark.parametrize("n_seqs,tiles,d", [(65, 40, 64), (100, 90, 64), (300, 200, 64), (300, 60, 128),
                                            (256, 130, 64), (257, 70, 128), (511, 40, 64)])
def test_many_ragged_sequences_in_parts(dev, n_seqs, tiles, d):
    """Four lengths a lane: sequences whose parts end anywhere in a lane's four, empty ones among them."""
    lens = np.random.default_rng(n_seqs).integers(0, 32 * tiles + 1, n_seqs)
    lens[[0, 5, 6, 63, 64, n_seqs - 1]] = [0, 32 * tiles, 1, 0, 32 * tiles - 1, 33]
    lens[np.random.default_rng(1).random(n_seqs) < 0.2] //= 100
    r = Round(dev, 61, 1, 2, d, 32, n_seqs, 32 * tiles)
    r.run(lens.tolist())


LINES = [  # hkv, group, d, page, tiles of each sequence: more than 16384 in all and 256 (64) an item as a mean
    (8, 2, 64, 64, [1500, 0, 3, 900, 1, 40]),
    (8, 5, 64, 32, [1, 1, 4000, 2]),
    (1, 4, 64, 128, [0, 20000, 0, 7, 31, 1, 2000]),
    (2, 3, 128, 64, [4000, 1, 0, 4300, 64, 2]),
    (8, 1, 128, 32, [300] * 3 + [1, 0, 900, 2, 600, 5]),
]


@pytest.mark.parametrize("hkv,group,d,page,tiles", LINES)
def test_a_ragged_line_of_few_sequences(dev, hkv, group, d, page, tiles):
    """Very long sequences beside empty ones and ones of a few tiles, whose stretches of the line one
    workgroup has several of."""
    lens = [max(0, 32 * n - (i * 7) % 32) for i, n in enumerate(tiles)]
    total = hkv * sum(max(1, -(-n // 32)) for n in lens)
    assert total > 16384 and total > (256 if d == 64 else 64) * hkv * len(lens)
    r = Round(dev, 62, hkv, group, d, page, len(lens), max(lens))
    r.run(lens)
    r.run(lens[::-1])


@pytest.mark.parametrize("n_seqs,hkv,tiles,d", [(70, 1, 700, 64), (90, 1, 420, 128), (200, 2, 150, 128)])
def test_a_ragged_line_of_many_sequences(dev, n_seqs, hkv, tiles, d):
    lens = np.random.default_rng(n_seqs).integers(0, 32 * tiles + 1, n_seqs)
    lens[[0, 9, 63, 64, n_seqs - 1]] = [0, 32 * tiles, 1, 0, 3]
    total = hkv * int(np.maximum(1, -(-lens // 32)).sum())
    assert total > 16384 and total > (256 if d == 64 else 64) * hkv * n_seqs
    r = Round(dev, 63, hkv, 2, d, 64, n_seqs, 32 * tiles)
    r.run(lens.tolist())


def test_ragged_lengths_that_change_under_a_graph(dev):
    """The sharing follows the lengths at each replay, not those of the capture."""
    r = Round(dev, 64, 2, 4, 64, 64, 6, 9000)
    q = r.x.q(6, 8)
    lens, qd = ints([9000] * 6, dev), up(q, dev)
    r.x.c.attn(0, qd, lens, table=r.table)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, out32 = r.x.c.attn(0, qd, lens, table=r.table, want_f32=True)
    for now in ([9000, 0, 1, 4500, 33, 8999], [0] * 6, [1] * 6, [0, 0, 0, 9000, 0, 0], [31, 32, 33, 64, 65, 1024]):
        lens.copy_(torch.tensor(now, dtype=torch.int32))
        g.replay()
        torch.cuda.synchronize()
        want, bound = (np.stack(y) for y in zip(*(r.want(q[b].astype(np.float64), n, 0.125)
                                                  for b, n in enumerate(now))))
        check(out, out32, want, bound)
        assert torch.equal(r.x.c.attn(0, qd, lens, table=r.table), out)
