"""The paged 4-bit K/V cache in numpy: its bytes from the written format, one position and channel at a
time where speed allows, attention and page scores in float64, and the page bookkeeping on Python
lists. Nothing here comes from the kernels."""

from __future__ import annotations

import numpy as np


def bf16_bits(x):
    """float32 -> bf16 bits, round to nearest even."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def bf16_f32(b):
    return (np.asarray(b, np.uint16).astype(np.uint32) << 16).view(np.float32)


def quant(x):
    """bf16 rows as float32 [..., D] -> codes uint8 [..., D], bits of d and of m [..., D/32]."""
    x = np.asarray(x, np.float32)
    g = x.reshape(*x.shape[:-1], -1, 32)
    bad = ~np.isfinite(g).all(-1)
    safe = np.where(bad[..., None], np.float32(0), g)
    lo, hi = safe.min(-1), safe.max(-1)
    with np.errstate(over="ignore", divide="ignore", invalid="ignore"):
        d = bf16_f32(bf16_bits((hi - lo) / np.float32(15)))
        bad |= ~np.isfinite(d)
        codes = np.clip(np.rint((safe - lo[..., None]) / d[..., None]), 0, 15)
    codes = np.where((d > 0)[..., None] & ~bad[..., None], codes, 0).astype(np.uint8)
    db = np.where(bad, 0x7FC0, bf16_bits(d)).astype(np.uint16)
    mb = np.where(bad, 0x7FC0, bf16_bits(lo)).astype(np.uint16)
    return codes.reshape(x.shape), db, mb


def places(d):
    """For K and V: byte offset in a tile and nibble (0 low, 1 high) of (position, channel)."""
    out = []
    for kind in "kv":
        byte, nib = np.empty((32, d), np.int64), np.empty((32, d), np.int64)
        for p in range(32):
            for ch in range(d):
                c = ch // 64
                if kind == "k":
                    tt, n = p // 16, p % 16
                    g, kg, i = (ch % 64) // 32, (ch % 32) // 8, ch % 8
                    dword, e = 2 * tt + g, [0, 2, 4, 6, 1, 3, 5, 7].index(i)
                else:
                    t, n = (ch % 64) // 16, ch % 16
                    kg, dword = (p % 16) // 4, t
                    e = p % 4 + 4 * (p // 16)
                lane = 16 * kg + n
                byte[p, ch] = (0 if kind == "k" else 16 * d) + (c * 64 + lane) * 16 + dword * 4 + e // 2
                nib[p, ch] = e % 2
        out.append((byte, nib))
    return out


_places: dict = {}


class Pages:
    """A pool of one layer as numpy bytes [n_pages, page bytes]."""

    def __init__(self, pool, hkv, d, page):
        self.pool, self.hkv, self.d, self.page = pool, hkv, d, page
        self.hb = page // 32 * 40 * d + 4 * d
        assert pool.shape[1] == hkv * self.hb
        self.kp, self.vp = _places.setdefault(d, places(d))

    def _at(self, head, p):
        return head * self.hb + p // 32 * 40 * self.d

    def write(self, page, head, p, k, v):
        """Rows k, v (float32 of bf16 values) at position p of a page."""
        d, t, base = self.d, p % 32, self._at(head, p)
        row = self.pool[page]
        for side, (x, (byte, nib)) in enumerate(((k, self.kp), (v, self.vp))):
            codes, db, mb = quant(x)
            at, hi = base + byte[t], nib[t]
            for half in (0, 1):
                w = hi == half
                keep = 0x0F if half else 0xF0
                row[at[w]] = (row[at[w]] & keep) | (codes[w] << (4 * half))
            s = base + 32 * d + side * 4 * d + t * (d // 32) * 4
            row[s:s + d // 8] = np.stack((db, mb), -1).astype("<u2").reshape(-1).view(np.uint8)

    def bounds(self, page, head):
        """(lo, hi) as a writable uint16 view [2, d]."""
        at = head * self.hb + self.page // 32 * 40 * self.d
        return self.pool[page, at:at + 4 * self.d].view("<u2").reshape(2, self.d)

    def append(self, table, pos, rows, k, v):
        """rows[b]: indices into k, v [N, hkv, d] written at pos[b], pos[b] + 1, .."""
        cap = table.shape[1] * self.page
        for b, idx in enumerate(rows):
            seen = {}
            for i, r in enumerate(idx):
                p = int(pos[b]) + i
                if not 0 <= p < cap:
                    continue
                pg = int(table[b, p // self.page])
                if not 0 <= pg < len(self.pool):
                    continue
                seen.setdefault((pg, p // self.page), []).append((p % self.page, r))
            for (pg, _), items in seen.items():
                for h in range(self.hkv):
                    for p, r in items:
                        self.write(pg, h, p, k[r, h], v[r, h])
                    x = np.stack([k[r, h] for _, r in items])
                    g = x.reshape(len(items), -1, 32)
                    with np.errstate(over="ignore", invalid="ignore"):
                        span = (g.max(-1) - g.min(-1)) / np.float32(15)
                        bad = ~np.isfinite(g).all(-1) | ~np.isfinite(bf16_f32(bf16_bits(span)))
                    poison = np.repeat(bad.any(0), 32)
                    lo, hi = x.min(0), x.max(0)
                    lo, hi = (np.where(poison, np.nan, y).astype(np.float32) for y in (lo, hi))
                    old = self.bounds(pg, h)
                    if items[0][0] != 0:
                        lo = np.minimum(lo, bf16_f32(old[0]))   # a NaN stays
                        hi = np.maximum(hi, bf16_f32(old[1]))
                    old[0], old[1] = bf16_bits_nan(lo), bf16_bits_nan(hi)

    def values(self, page, head, p):
        """What K and V of a position stand for (float32, one rounding of d * code + m)."""
        d, t, base = self.d, p % 32, self._at(head, p)
        row, out = self.pool[page], []
        for side, (byte, nib) in enumerate((self.kp, self.vp)):
            codes = (row[base + byte[t]] >> (4 * nib[t])) & 15
            s = base + 32 * d + side * 4 * d + t * (d // 32) * 4
            dm = bf16_f32(row[s:s + d // 8].view("<u2")).reshape(-1, 2).astype(np.float64)
            with np.errstate(invalid="ignore"):
                out.append((codes.reshape(-1, 32) * dm[:, :1] + dm[:, 1:]).reshape(-1).astype(np.float32))
        return out

    def scales(self, page, head, p):
        """d and |m| of a position's groups for K and V, float64 [2, d/32] each."""
        d, t, base = self.d, p % 32, self._at(head, p)
        s = base + 32 * d + t * (d // 32) * 4
        two = [bf16_f32(self.pool[page][s + o:s + o + d // 8].view("<u2")).reshape(-1, 2)
               for o in (0, 4 * d)]
        return np.stack([x[:, 0] for x in two]).astype(np.float64), \
            np.abs(np.stack([x[:, 1] for x in two])).astype(np.float64)


def bf16_bits_nan(x):
    return np.where(np.isnan(x), 0x7FC0, bf16_bits(np.where(np.isnan(x), 0, x))).astype(np.uint16)


def attention(pages: Pages, table, q, ends, scale, keep=None):
    """One sequence and kv head at a time: q [rows, heads, d] float64 of sequence with table row
    `table`, row i seeing positions [0, ends[i]) of kv head h = head // group. keep: per kv head a set
    of logical pages. Returns (out, bound) float64 [rows, heads, d]: bound is how far an fp32
    computation through the codes may be off."""
    rows, heads, d = q.shape
    group = heads // pages.hkv
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    cap = len(table) * pages.page
    top = max([0] + [min(int(e), cap) for e in ends])
    for h in range(pages.hkv):
        pos = [p for p in range(top) if keep is None or p // pages.page in keep[h]]
        kv = [pages.values(table[p // pages.page], h, p % pages.page) for p in pos]
        sc = [pages.scales(table[p // pages.page], h, p % pages.page) for p in pos]
        if not kv:
            continue
        k = np.stack([x for x, _ in kv]).astype(np.float64)
        v = np.stack([x for _, x in kv]).astype(np.float64)
        dk, mk = (np.repeat(np.stack([s[i][0] for s in sc]), 32, -1) for i in (0, 1))
        dv, mv = (np.repeat(np.stack([s[i][1] for s in sc]), 32, -1) for i in (0, 1))
        at = np.array(pos)
        for i in range(rows):
            see = at < ends[i]
            if not see.any():
                continue
            for g in range(group):
                x = q[i, h * group + g]
                s = scale * (k[see] @ x)
                p = np.exp(s - s.max()) if np.isfinite(s).all() else np.full(s.shape, np.nan)
                p = p / p.sum()
                out[i, h * group + g] = p @ v[see]
                # scores: 32 products and sums of up to 143 d |q| and m |q| a group, each to 2^-24, and
                # the exponent's own rounding; values: p d in two bf16 terms (2^-18 of a code of up to
                # 31), and sums of up to 31 p d over the tiles, joined over at most 64 splits of 4 waves;
                # blocks: k, v and p are two bf16 terms each, 2^-18 of them left out
                es = (abs(scale) * ((143 * dk[see] + mk[see]) @ np.abs(x)) * 40 + 4 * np.abs(s)) * 2.0 ** -24
                es += abs(scale) * ((15 * dk[see] + mk[see]) @ np.abs(x)) * 2.0 ** -18
                tiles = len(pos) / 32 + 80
                bound[i, h * group + g] = (2 * es.max() + 2.0 ** -20 + 3 * 2.0 ** -18) * (p @ (15 * dv[see] + mv[see])) \
                    + (p @ dv[see]) * (31 * 2.0 ** -18 + 31 * tiles * 2.0 ** -24) \
                    + (p @ mv[see]) * tiles * 2.0 ** -24
    return out, bound


def select(pages: Pages, table, q, length, n_sel, n_first, n_last):
    """The pages of one sequence: q [heads, d] float64 -> [hkv, n_sel]."""
    heads, d = q.shape
    group, n = heads // pages.hkv, -(-length // pages.page)
    out = np.full((pages.hkv, n_sel), -1, np.int32)
    for h in range(pages.hkv):
        key = []
        for p in range(n):
            lo, hi = (bf16_f32(x).astype(np.float64) for x in pages.bounds(table[p], h))
            x = q[h * group:(h + 1) * group]
            s = np.maximum(x * lo, x * hi).sum()
            rank = 2 if p < n_first or p >= n - n_last else 1 if np.isnan(s) else 0
            key.append((-rank, -s if rank == 0 else 0.0, p))
        best = sorted(k[2] for k in sorted(key)[:n_sel])
        out[h, :len(best)] = best
    return out


class Book:
    """The bookkeeping: a table of lists, counts, lengths; `moves` collects page copies (from, to)."""

    def __init__(self, n_seqs, table_len, n_pages, page):
        self.table = np.full((n_seqs, table_len), -1, np.int32)
        self.lens = np.zeros(n_seqs, np.int32)
        self.refs = np.zeros(n_pages, np.int32)
        self.page = page
        self.moves = []

    def _free(self):
        return [p for p in range(len(self.refs)) if self.refs[p] == 0]

    def reserve(self, want):
        free, bad, dry = self._free(), 0, False
        for b, w in enumerate(want):
            need = -(-max(0, int(w)) // self.page)
            have = int((self.table[b] >= 0).sum())
            if need > self.table.shape[1]:
                bad += 1
                continue
            if need <= have:
                continue
            if dry or need - have > len(free):
                bad, dry = bad + 1, True
                continue
            for j in range(have, need):
                self.table[b, j] = free.pop(0)
                self.refs[self.table[b, j]] = 1
        return bad

    def fork(self, src, dst):
        free, bad, n = self._free(), 0, len(self.lens)
        inside = [0 <= s < n and 0 <= d < n for s, d in zip(src, dst)]
        sources = {s for s, ok in zip(src, inside) if ok}
        took = set()
        for s, d, ok in zip(src, dst, inside):
            if not ok:
                bad += 1
                continue
            first = d not in took
            took.add(d)
            if not first or d in sources or self.table[d, 0] >= 0:
                bad += 1
                continue
            length = int(self.lens[s])
            full, rest = divmod(length, self.page)
            if length and not 0 <= self.table[s, (length - 1) // self.page] < len(self.refs):
                bad += 1
                continue
            if rest and not free:
                bad += 1
                continue
            self.table[d] = -1
            self.table[d, :full] = self.table[s, :full]
            for p in self.table[d, :full]:
                self.refs[p] += 1
            if rest:
                self.table[d, full] = free.pop(0)
                self.refs[self.table[d, full]] = 1
                self.moves.append((int(self.table[s, full]), int(self.table[d, full])))
            self.lens[d] = self.lens[s]
        return bad

    def free(self, seqs):
        bad = 0
        for s in seqs:
            if not 0 <= s < len(self.lens):
                bad += 1
                continue
            for p in self.table[s][self.table[s] >= 0]:
                self.refs[p] -= 1
            self.table[s], self.lens[s] = -1, 0
        return bad

    def compact(self):
        live = int((self.refs > 0).sum())
        holes = [p for p in range(live) if self.refs[p] == 0]
        movers = [p for p in range(live, len(self.refs)) if self.refs[p] > 0]
        for a, z in zip(movers, holes):
            self.moves.append((a, z))
            self.table[self.table == a] = z
            self.refs[z], self.refs[a] = self.refs[a], 0
        return live
