"""Attention over shared prefixes against float64, and a run of it in a graph."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def rows(g, *shape):
    return torch.randn(shape, device="cuda", generator=g).to(torch.bfloat16)


def reference(q, kp, vp, plens, k, v, lens, groups, scale):
    """float64 attention, and the largest sum |p v| of a row's channels (what roundings of p scale with)."""
    b, hq, d = q.shape
    hkv = k.shape[1]
    g = hq // hkv
    out = torch.zeros((b, hq, d), dtype=torch.float64, device=q.device)
    mag = torch.zeros_like(out)
    for i in range(b):
        p = next((x for x, (lo, hi) in enumerate(groups) if lo <= i < hi), None)
        for h in range(hkv):
            n = max(int(lens[i]), 0)
            kk, vv = k[i, h, :n].double(), v[i, h, :n].double()
            if p is not None:
                m = max(int(plens[p]), 0)
                kk, vv = torch.cat((kp[p, h, :m].double(), kk)), torch.cat((vp[p, h, :m].double(), vv))
            if len(kk):
                w = torch.softmax(q[i, h * g:(h + 1) * g].double() @ kk.T * scale, -1)
                out[i, h * g:(h + 1) * g], mag[i, h * g:(h + 1) * g] = w @ vv, w @ vv.abs()
    return out, mag


def check(got, f32, want, mag):
    """A weight is its upper half, which leaves up to 2^-7 of it, and that rounded to bf16: 2^-15 at most is
    lost, of the sum that divides likewise; a score's scaled value (below 2^6) is rounded a few times in
    fp32, 2^-24 * 2^6 each, and so are the sums."""
    err = (f32.double() - want).abs()
    assert bool((err <= 2.0 ** -13 * mag + 1e-30).all()), float((err / (mag + 1e-30)).max())
    assert torch.equal(got, f32.to(torch.bfloat16))


CASES = [
    # b, groups, hq, hkv, d, plens, lens
    (1, [(0, 1)], 8, 8, 64, [1], [0]),
    (1, [(0, 1)], 16, 1, 128, [130], [1]),
    (2, [(0, 2)], 40, 8, 64, [513], [33, 1]),
    (3, [(0, 3)], 10, 2, 64, [64], [0, 129, 64]),
    (8, [(0, 8)], 40, 8, 64, [2048], [128, 5, 77, 1, 0, 64, 63, 65]),
    (5, [(0, 2), (2, 2), (2, 5)], 14, 2, 128, [300, 50, 999], [7, 300, 0, 1, 31]),
    (6, [(1, 4)], 8, 1, 64, [777], [3, 0, 12, 500, 0, 9]),            # sequences without a prefix
    (4, [(0, 2), (2, 4)], 4, 2, 64, [0, 65], [0, 3, 2, 0]),            # an empty prefix: one row sees nothing
    (33, [(0, 33)], 7, 1, 64, [4097], [i * 3 for i in range(33)]),
    (20, [(0, 9), (9, 20)], 32, 4, 128, [1025, 320], [i for i in range(20)]),
    (70, [(i, i + 1) for i in range(70)], 4, 2, 64, [i * 5 for i in range(70)], [i % 7 for i in range(70)]),
    (3, [(0, 3)], 16, 1, 64, [40000], [1, 2, 3000]),
    # two and five workgroups a compute unit
    (64, [(0, 20), (20, 64)], 40, 8, 64, [300, 401], [i % 41 for i in range(64)]),
    (300, [(0, 300)], 16, 4, 128, [60], [i % 40 for i in range(300)]),
]


@pytest.mark.parametrize("case", CASES, ids=[f"b{c[0]}p{len(c[1])}hq{c[2]}_{c[3]}d{c[4]}" for c in CASES])
def test_prefix_decode(dev, case):
    from llmnputest_amd import ops
    b, groups, hq, hkv, d, plens, lens = case
    g = torch.Generator(device="cuda").manual_seed(len(plens) * 100 + b)
    lp, lo = max(plens) + 3, max(lens) + 2
    kp, vp, k, v = (rows(g, n, hkv, m, d) for n, m in ((len(plens), lp), (len(plens), lp), (b, lo), (b, lo)))
    for i, n in enumerate(plens):   # what lies behind the lengths must not be seen
        kp[i, :, n:], vp[i, :, n:] = float("nan"), float("inf")
    for i, n in enumerate(lens):
        k[i, :, n:], v[i, :, n:] = float("inf"), float("nan")
    q = rows(g, b, hq, d) * 1.5
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    cu = None if groups == [(0, b)] else ints([groups[0][0]] + [hi for _, hi in groups])
    out, f32 = ops.gqa_prefix_decode(q, kp, vp, ints(plens), k, v, ints(lens), cu=cu, want_f32=True)
    want, mag = reference(q, kp, vp, plens, k, v, lens, groups, d ** -0.5)
    check(out, f32, want, mag)
    again = ops.gqa_prefix_decode(q, kp, vp, ints(plens), k, v, ints(lens), cu=cu)
    assert torch.equal(out, again)   # no order of arrival in it


@pytest.mark.parametrize("b", [2, 20])
def test_scores_that_rise(dev, b):
    """Maxima that move late and far, by more than 2^8 at once and by little; scores of -inf and then far below
    zero; rows of one workgroup that differ in all of that."""
    from llmnputest_amd import ops
    g = torch.Generator(device="cuda").manual_seed(b)
    n, d = 3000, 64
    kp, vp = rows(g, 1, 2, n, d), rows(g, 1, 2, n, d)
    kp[0, 0] *= torch.linspace(0.1, 3, n, device="cuda")[:, None]
    kp[0, 0, 2500] *= 8
    kp[0, 1, :200, 0] = float("-inf")          # -inf for every q whose first channel is positive
    kp[0, 1, 200:, 0] = -300.0
    q = rows(g, b, 8, d)
    q[..., 0] = q[..., 0].abs() + 0.5
    q[1] *= 0.01
    none = torch.zeros((b, 2, 0, d), dtype=torch.bfloat16, device="cuda")
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    out, f32 = ops.gqa_prefix_decode(q, kp, vp, ints([n]), none, none, ints([0] * b), want_f32=True)
    want, mag = reference(q, kp, vp, [n], none, none, [0] * b, [(0, b)], d ** -0.5)
    # scores reach 2^9 here: 2^-24 of that, a few times, in the exponent
    assert bool(((f32.double() - want).abs() <= 2.0 ** -11 * mag + 1e-30).all())
    assert torch.equal(out, f32.to(torch.bfloat16))


@pytest.mark.parametrize("b", [1, 30])
def test_nan_stays(dev, b):
    """A NaN or an infinity of a key or a value that a row sees shows in it, and in no other group's rows."""
    from llmnputest_amd import ops
    g = torch.Generator(device="cuda").manual_seed(7)
    kp, vp = rows(g, 2, 1, 1500, 64), rows(g, 2, 1, 1500, 64)
    kp[0, 0, 900, 3] = float("nan")
    vp[1, 0, 1400, 5] = float("inf")
    q, k, v = rows(g, 2 * b, 4, 64), rows(g, 2 * b, 1, 3, 64), rows(g, 2 * b, 1, 3, 64)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    out = ops.gqa_prefix_decode(q, kp, vp, ints([1500, 1500]), k, v, ints([3] * (2 * b)), cu=ints([0, b, 2 * b]))
    assert bool(out[:b].isnan().all())
    bad = ~out[b:].isfinite()
    assert bool(bad[..., 5].all()) and not bool(bad[..., :5].any()) and not bool(bad[..., 6:].any())


@pytest.mark.parametrize("d", [64, 128])
def test_more_prefixes_than_sequences(dev, d):
    """The first sequences of a larger batch: prefixes without members, before, between and behind theirs."""
    from llmnputest_amd import ops
    g = torch.Generator(device="cuda").manual_seed(d)
    plens, edges = [1100 + 7 * i for i in range(70)], [0, 0, 0, 2] + [2] * 60 + [6, 9, 30, 31, 32, 33, 40]
    kp, vp = rows(g, 70, 2, max(plens), d), rows(g, 70, 2, max(plens), d)
    lens = [0, 3, 9, 140, 1, 2, 5]
    k, v, q = rows(g, 7, 2, 140, d), rows(g, 7, 2, 140, d), rows(g, 7, 8, d)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    want, mag = reference(q, kp, vp, plens, k, v, lens, list(zip(edges, edges[1:])), d ** -0.5)
    for b in (7, 1):
        out, f32 = ops.gqa_prefix_decode(q[:b], kp, vp, ints(plens), k[:b], v[:b], ints(lens[:b]), cu=ints(edges),
                                         want_f32=True)
        check(out, f32, want[:b], mag[:b])
