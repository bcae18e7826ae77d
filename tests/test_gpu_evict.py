"""Attention that sums its weights, and eviction by them, against float64."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def rows(g, *shape):
    return torch.randn(shape, device="cuda", generator=g).to(torch.bfloat16)


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def reference(q, k, v, lens, scale):
    """float64: outputs, sums of |p v|, and what each position is given."""
    b, hq, d = q.shape
    hkv, n = k.shape[1:3]
    g = hq // hkv
    out = torch.zeros((b, hq, d), dtype=torch.float64, device=q.device)
    mag, given = torch.zeros_like(out), torch.zeros((b, hkv, n), dtype=torch.float64, device=q.device)
    for i in range(b):
        m = min(max(int(lens[i]), 0), n)
        if m == 0:
            continue
        for h in range(hkv):
            w = torch.softmax(q[i, h * g:(h + 1) * g].double() @ k[i, h, :m].double().T * scale, -1)
            out[i, h * g:(h + 1) * g] = w @ v[i, h, :m].double()
            mag[i, h * g:(h + 1) * g] = w @ v[i, h, :m].double().abs()
            given[i, h, :m] = w.sum(0)
    return out, mag, given


# a score's scaled value (below 2^6 here) is rounded a few times in fp32, 2^-24 * 2^6 each, and so is its
# exponential, the sum and its reciprocal: below 2^-16 of a weight together
WEIGHT = 2.0 ** -16
# the outputs' weights enter with 17 bits
OUT = 2.0 ** -15

CASES = [
    (1, 8, 8, 64, [1]),
    (2, 40, 8, 64, [513, 1]),
    (3, 16, 1, 128, [129, 0, 1000]),
    (4, 6, 2, 64, [0, 128, 127, 2500]),
    (8, 40, 8, 64, [2176, 30, 700, 1, 2048, 255, 256, 257]),
    (2, 14, 2, 128, [9000, 8191]),
    (1, 5, 1, 64, [70000]),
    (300, 4, 4, 64, [i * 2 for i in range(300)]),
    # many rows: with their scores in LDS as far as it holds them, in memory beyond
    (24, 40, 8, 64, [max(2500 - 113 * i, 0) for i in range(24)]),
    (160, 3, 1, 128, [(i * 37) % 1100 for i in range(160)]),
    (40, 64, 4, 64, [(i * 101) % 900 for i in range(40)]),
    (12, 4, 2, 128, [600 - 50 * i for i in range(12)]),
]


@pytest.mark.parametrize("case", CASES, ids=[f"b{c[0]}hq{c[1]}_{c[2]}d{c[3]}l{max(c[4])}" for c in CASES])
def test_decode_weights(dev, case):
    from llmnputest_amd import ops
    b, hq, hkv, d, lens = case
    g = torch.Generator(device="cuda").manual_seed(b + hq)
    n = max(lens) + 3
    k, v = rows(g, b, hkv, n, d), rows(g, b, hkv, n, d)
    for i, m in enumerate(lens):
        k[i, :, m:], v[i, :, m:] = float("nan"), float("nan")
    q = rows(g, b, hq, d)
    weights = torch.full((b, hkv, n), 7.0, device="cuda")
    total = torch.zeros((b, hkv, n), dtype=torch.float64, device="cuda")
    for step, start in ((0, True), (1, False), (2, False)):
        q = rows(g, b, hq, d)
        at = [max(m - 2 + step, 0) if m else 0 for m in lens]     # lengths grow to theirs
        out, f32 = ops.gqa_decode_weights(q, k, v, ints(at), weights, start=start, want_f32=True)
        want, mag, given = reference(q, k, v, at, d ** -0.5)
        assert bool(((f32.double() - want).abs() <= OUT * mag + 1e-30).all())
        assert torch.equal(out, f32.to(torch.bfloat16))
        total += given
        seen = torch.arange(n, device="cuda") < ints(at)[:, None, None]
        err = (weights.double() - total).abs()
        assert bool((err <= WEIGHT * total + 1e-30)[seen.expand_as(err)].all())
        assert bool((weights == 7.0)[~seen.expand_as(err)].all())   # behind the newest nothing is written
    assert bool(((weights.double().sum(-1) - total.sum(-1)).abs()[[m > 2 for m in lens]] < 21 * n).all())


def evict_reference(k, v, w, lens, budget, recent, theta):
    """What is kept, K turned in float64."""
    b, hkv, n, d = k.shape
    kept = torch.full((b, hkv, budget), -1, dtype=torch.int64)
    ks = [[None] * hkv for _ in range(b)]
    for i in range(b):
        m = min(max(lens[i], 0), n)
        for h in range(hkv):
            x = w[i, h, :m].double()
            x = torch.where(x.isnan(), float("inf"), x).tolist()
            nan = w[i, h, :m].isnan().tolist()
            best = list(range(m))
            if m > budget:
                old = sorted(range(m - recent), key=lambda p: (not nan[p], -x[p], p))[:budget - recent]
                best = sorted(old) + list(range(m - recent, m))
            kept[i, h, :len(best)] = torch.tensor(best, dtype=torch.int64)
            at = torch.tensor(best, dtype=torch.int64, device=k.device)
            kk = k[i, h, at].double()
            if theta:
                by = (torch.arange(len(best), device=k.device) - at).double()[:, None]
                by = by * theta ** (-2 * torch.arange(d // 2, device=k.device).double() / d)
                lo, hi = kk[:, :d // 2], kk[:, d // 2:]
                kk = torch.cat((lo * by.cos() - hi * by.sin(), hi * by.cos() + lo * by.sin()), -1)
            ks[i][h] = kk
    return kept, ks


EVICT = [
    # b, hkv, d, lens, budget, recent, turn, kind of weights
    (1, 1, 64, [1], 1, 0, False, "random"),
    (1, 2, 64, [5], 1, 1, True, "random"),
    (2, 3, 128, [100, 40], 64, 16, True, "random"),
    (3, 8, 64, [1000, 0, 513], 512, 64, True, "random"),
    (2, 2, 64, [3000, 2999], 1000, 0, False, "equal"),
    (2, 2, 64, [5000, 3000], 700, 700, True, "random"),
    (2, 1, 64, [4097, 1025], 1024, 100, True, "special"),
    (1, 2, 128, [40000], 5000, 333, True, "random"),
    (4, 2, 64, [2049, 2048, 2047, 1], 2048, 5, True, "steps"),
    # around the most positions whose keys one workgroup holds (room for two more than the longest)
    (2, 2, 64, [16382, 9000], 3000, 100, True, "steps"),
    (1, 2, 64, [16382], 700, 50, False, "special"),
    (2, 2, 128, [6001, 4098], 1000, 3, True, "equal"),
    (2, 2, 128, [16383, 50], 1000, 77, True, "random"),
    (3, 1, 64, [20000, 4096, 300], 600, 17, True, "special"),
    (2, 2, 64, [30000, 12289], 9000, 0, False, "equal"),
]


@pytest.mark.parametrize("place", ["in place", "into"])
@pytest.mark.parametrize("case", EVICT, ids=[f"b{c[0]}h{c[1]}d{c[2]}l{max(c[3])}k{c[4]}r{c[5]}{c[7]}" for c in EVICT])
def test_evict(dev, case, place):
    from llmnputest_amd import ops
    b, hkv, d, lens, budget, recent, turn, kind = case
    g = torch.Generator(device="cuda").manual_seed(budget + recent)
    n = max(lens) + 2
    k, v = rows(g, b, hkv, n, d), rows(g, b, hkv, n, d)
    w = torch.exp(2 * torch.randn((b, hkv, n), device="cuda", generator=g))
    if kind == "equal":
        w = torch.ones_like(w)
    elif kind == "steps":
        w = torch.randint(0, 4, w.shape, device="cuda", generator=g).float()
    elif kind == "special":
        x = torch.randint(0, 7, w.shape, device="cuda", generator=g)
        for i, val in enumerate((float("nan"), float("inf"), 0.0, -0.0, -1.0)):
            w = torch.where(x == i, val, w)
    table = ops.rope_table(n, d) if turn else None
    kept, ks = evict_reference(k, v, w, lens, budget, recent, 10000.0 if turn else 0)
    room = n if place == "in place" else budget + 5
    if place == "in place":
        k2, v2, w2, l2 = k.clone(), v.clone(), w.clone(), ints(lens)
        got = ops.kv_evict(k2, v2, w2, l2, budget, recent, rope=table)
    else:
        k2, v2 = (torch.full((b, hkv, room, d), 3.0, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        w2, l2 = torch.full((b, hkv, room), 3.0, device="cuda"), ints([9] * b)
        k0, v0, w0 = k.clone(), v.clone(), w.clone()
        got = ops.kv_evict(k, v, w, ints(lens), budget, recent, rope=table, into=(k2, v2, w2, l2))
        assert torch.equal(k, k0) and torch.equal(v, v0) and torch.equal(w.view(torch.int32), w0.view(torch.int32))
    assert torch.equal(got.cpu().long(), kept)
    ends = [min(m, budget) for m in lens]
    assert l2.tolist() == ends
    for i in range(b):
        m = ends[i]
        for h in range(hkv):
            at = kept[i, h, :m].cuda()
            assert torch.equal(v2[i, h, :m], v[i, h, at])
            assert torch.equal(w2[i, h, :m].view(torch.int32), w[i, h, at].view(torch.int32))
            # cos and sin rounded to fp32, two products and a sum in fp32, then half a step of bf16
            size = (k[i, h, at].double().abs().view(m, 2, d // 2).sum(1)).repeat(1, 2)
            assert bool(((k2[i, h, :m].double() - ks[i][h]).abs() <= 2.0 ** -8 * ks[i][h].abs() + 2.0 ** -21 * size).all())
            still = at == torch.arange(m, device="cuda")
            assert torch.equal(k2[i, h, :m][still], k[i, h, at][still])
            if place == "into":
                assert bool((w2[i, h, m:] == 0).all())
                assert bool((k2[i, h, m:] == 3).all()) and bool((v2[i, h, m:] == 3).all())
            else:
                assert bool((w2[i, h, m:lens[i]] == 0).all())
                assert torch.equal(k2[i, h, max(m, 0):], k[i, h, max(m, 0):]) and torch.equal(v2[i, h, m:], v[i, h, m:])
                assert torch.equal(w2[i, h, lens[i]:].view(torch.int32), w[i, h, lens[i]:].view(torch.int32))
