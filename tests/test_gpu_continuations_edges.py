"""Several continuations of a prompt, at the edges: what workgroups' waves share in LDS, scales of nothing,
signs of zero, and lengths that need another path than the usual ones."""

import pytest
import torch

from llmnputest_amd.granite import GraniteConfig, GraniteDecoder, GraniteWeights
from tests.test_gpu_evict import CASES as EVICT_CASES, WEIGHT
from tests.test_gpu_prefix import check, reference, rows

pytestmark = pytest.mark.gpu


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("b", [5, 8, 13, 40])
def test_first_tile_of_a_prefix_part(dev, b, d):
    """Parts of four tiles of 64 positions, the first of which has nearly all of the weight and the third, whose
    rows of K take its place in LDS, none of it; waves without query rows among those with some."""
    from llmnputest_amd import ops
    g = torch.Generator(device="cuda").manual_seed(b)
    hq, hkv, n = 40, 8, 3001
    u = torch.randn((hkv, 1, d), device="cuda", generator=g).sign()
    toward = torch.tensor([2.0, 0.0, -2.0, 0.0], device="cuda")[torch.arange(n, device="cuda") // 64 % 4]
    kp = (toward[:, None] * u + 0.1 * torch.randn((1, hkv, n, d), device="cuda", generator=g)).to(torch.bfloat16)
    vp = rows(g, 1, hkv, n, d)
    q = (u.expand(hkv, hq // hkv, d).reshape(hq, d) + 0.1 * torch.randn((b, hq, d), device="cuda", generator=g)).to(torch.bfloat16)
    k, v, lens = rows(g, b, hkv, 3, d), rows(g, b, hkv, 3, d), [i % 4 for i in range(b)]
    want, mag = reference(q, kp, vp, [n], k, v, lens, [(0, b)], d ** -0.5)
    first = None
    for _ in range(10):
        out, f32 = ops.gqa_prefix_decode(q, kp, vp, ints([n]), k, v, ints(lens), want_f32=True)
        check(out, f32, want, mag)
        first = f32 if first is None else first
        assert torch.equal(f32, first)


def test_graphs_keep_their_workspace(dev):
    """A decoder's graphs go on in the memory they were captured with, also when its workspace has grown since."""
    cfg = GraniteConfig(n_layers=2, vocab=4096)
    dec = GraniteDecoder(GraniteWeights.synthetic(cfg, seed=3, device="cuda"), 2, 256, track_weights=True)
    dec.seed_cache(150, seed=9)
    want, _ = dec.generate([3, 4], [150, 90], 20)
    size = dec.ws.buf.numel()
    dec.ws.get(2 * size)
    others = [torch.full((size,), 0x5A, dtype=torch.uint8, device="cuda") for _ in range(3)]
    dec.seed_cache(150, seed=9)
    got, _ = dec.generate([3, 4], [150, 90], 20)
    assert (got == want).all() and all(bool((x == 0x5A).all()) for x in others)
    assert dec.evict([170, 110], 100, 16) == [100, 100]
    got, _ = dec.generate([5, 6], [100, 100], 20)
    assert got.shape == (2, 20) and all(bool((x == 0x5A).all()) for x in others)


@pytest.mark.parametrize("scale", [0.0, 1e-46, 0.05])
@pytest.mark.parametrize("d", [64, 128])
def test_ends_of_prefixes(dev, d, scale):
    """Prefixes that end at every place of a tile, as rows of a wide product, and own rows; with a scale of nothing
    (or one that is nothing in fp32) the answer is the mean of what is seen."""
    from llmnputest_amd import ops
    g = torch.Generator(device="cuda").manual_seed(d)
    plens = [1, 5, 31, 32, 33, 47, 63, 64, 65, 95, 96, 97, 128, 129, 160, 193, 700, 1101]
    b = 2 * len(plens)
    groups = [(2 * i, 2 * i + 2) for i in range(len(plens))]
    lens = [(0, 3, 129, 40)[i % 4] for i in range(b)]
    kp, vp = rows(g, len(plens), 1, 1104, d), rows(g, len(plens), 1, 1104, d)
    k, v, q = rows(g, b, 1, 130, d), rows(g, b, 1, 130, d), rows(g, b, 16, d)
    for i, n in enumerate(plens):
        kp[i, :, n:], vp[i, :, n:] = float("nan"), float("inf")
    cu = ints([0] + [hi for _, hi in groups])
    out, f32 = ops.gqa_prefix_decode(q, kp, vp, ints(plens), k, v, ints(lens), cu=cu, scale=scale, want_f32=True)
    want, mag = reference(q, kp, vp, plens, k, v, lens, groups, scale)
    check(out, f32, want, mag)


def test_weights_without_a_scale(dev):
    """A scale of 0: every position is given the same."""
    from llmnputest_amd import ops
    g = torch.Generator(device="cuda").manual_seed(1)
    lens = [3000, 1, 77]
    k, v, q = rows(g, 3, 2, 3000, 64), rows(g, 3, 2, 3000, 64), rows(g, 3, 10, 64)
    w = torch.zeros((3, 2, 3000), device="cuda")
    out = ops.gqa_decode_weights(q, k, v, ints(lens), w, start=True, scale=0.0, want_f32=True)[1]
    for i, n in enumerate(lens):
        mean = v[i, :, :n].double().mean(1).repeat_interleave(5, 0)
        # equal weights are exact; sums of n terms and a quotient in fp32
        assert bool(((out[i].double() - mean).abs() <= 2.0 ** -15 * v[i, :, :n].double().abs().mean(1).repeat_interleave(5, 0)).all())
        assert torch.allclose(w[i, :, :n], torch.full_like(w[i, :, :n], 5 / n), rtol=2.0 ** -20, atol=0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("v", [9, 5000, 100352])
def test_zeros_are_one_value(dev, v, dtype):
    """0 and -0 tie, and the lowest token takes it, within a thread's tokens and across workgroups."""
    from llmnputest_amd import ops
    x = torch.full((4, v), -1.0, dtype=dtype, device="cuda")
    x[0, 3], x[0, v - 1] = -0.0, 0.0
    x[1, 3], x[1, v - 1] = 0.0, -0.0
    x[2, 5], x[2, 6], x[2, 7] = -0.0, -0.0, 0.0
    x[3, v - 2], x[3, v - 1] = -0.0, 2.0 ** -126
    keys = torch.empty(4, dtype=torch.int64, device="cuda")
    out, token = ops.adjust_logits(x, keys=keys)
    assert token.tolist() == [3, 3, 5, v - 1]
    assert (0xFFFFFFFF - (keys & 0xFFFFFFFF)).tolist() == token.tolist()
    assert torch.equal(out.view(torch.int16), x.view(torch.int16))   # the logits' own zeros stay as they are


def test_biases_are_summed_first(dev):
    """A token that is listed twice gets the sum of its biases: 1 + (2^24 - 2^24), not (1 + 2^24) - 2^24."""
    from llmnputest_amd import ops
    big = 2.0 ** 24
    x = torch.ones((2, 40), device="cuda")
    bias = (ints([7, 9, 7, 39, 39, 39]), torch.tensor([big, 0.5, -big, big, 1.0, -big], device="cuda"), ints([0, 3, 6]))
    out, token = ops.adjust_logits(x, bias=bias)
    want = torch.ones((2, 40), device="cuda")
    want[0, 9] = 1.5                  # 39: big + 1 is big in fp32, so its sum is 0
    assert torch.equal(out, want) and token.tolist() == [9, 0]


@pytest.mark.parametrize("case", EVICT_CASES, ids=[f"b{c[0]}hq{c[1]}_{c[2]}d{c[3]}l{max(c[4])}" for c in EVICT_CASES])
def test_weights_add_up(dev, case):
    """What a step gives the positions of a kv head is one for each of its query heads, all together; what lies
    behind the newest is no part of it."""
    from llmnputest_amd import ops
    b, hq, hkv, d, lens = case
    g = torch.Generator(device="cuda").manual_seed(hq)
    n = max(lens) + 3
    k, v = rows(g, b, hkv, n, d), rows(g, b, hkv, n, d)
    weights = torch.full((b, hkv, n), 7.0, device="cuda")
    seen = torch.arange(n, device="cuda") < ints(lens)[:, None, None]
    for step in range(3):
        # the last position is the newest each time: what it was given before is gone
        before = weights.double()
        ops.gqa_decode_weights(rows(g, b, hq, d), k, v, ints(lens), weights, start=step == 0)
        newest = torch.stack([before[i, :, max(m - 1, 0)] * (m > 0) for i, m in enumerate(lens)])
        was = torch.where(seen, before, 0.0).sum(-1) - newest if step else torch.zeros_like(newest)
        now = torch.where(seen, weights.double(), 0.0).sum(-1)
        want = hq // hkv * (ints(lens)[:, None] > 0).double().expand_as(now)
        # each weight within WEIGHT of itself; what was there before is rounded once more by the addition
        assert bool(((now - was - want).abs() <= WEIGHT * want + 2.0 ** -24 * was).all())
        assert bool((weights == 7.0)[~seen.expand_as(weights)].all())


@pytest.mark.parametrize("b,hkv,n,budget,recent", [(16400, 1, 21, 9, 2), (2050, 8, 16390, 40, 7)])
def test_more_caches_than_counters(dev, b, hkv, n, budget, recent):
    """More sequences, or (sequence, kv head)s, than a workspace has counters: a workgroup selects alone, also from
    more positions than its registers hold."""
    from llmnputest_amd import ops
    g = torch.Generator(device="cuda").manual_seed(n)
    k = torch.empty((b, hkv, n, 64), dtype=torch.bfloat16, device="cuda")
    k.copy_((torch.arange(n, device="cuda") % 251)[:, None].expand(n, 64).to(torch.bfloat16))
    w = torch.randint(0, 1000, (b, hkv, n), device="cuda", generator=g).float()
    lens = [n - 3 * (i % 5) for i in range(b)]
    into = tuple(torch.zeros(s, dtype=t, device="cuda") for s, t in (
        ((b, hkv, budget, 64), torch.bfloat16), ((b, hkv, budget, 64), torch.bfloat16), ((b, hkv, budget), torch.float32), ((b,), torch.int32)))
    kept = ops.kv_evict(k, k.view_as(k), w, ints(lens), budget, recent, into=into).long()
    assert into[3].tolist() == [budget] * b
    index = torch.arange(n, device="cuda")
    for i0 in range(0, b, 512):
        m, x = ints(lens[i0:i0 + 512])[:, None, None], w[i0:i0 + 512]
        x = torch.where(index < m - recent, x, torch.where(index < m, float("inf"), float("-inf")))
        want = torch.sort(x, descending=True, stable=True).indices[..., :budget].sort(-1).values
        assert torch.equal(kept[i0:i0 + 512], want)
        assert torch.equal(into[2][i0:i0 + 512], torch.gather(w[i0:i0 + 512], 2, want))
        for to in into[:2]:
            assert torch.equal(to[i0:i0 + 512], (want % 251).to(torch.bfloat16)[..., None].expand(*want.shape, 64))
