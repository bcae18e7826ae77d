"""Counts of tokens and the rules for the next one against the steps in float64 and float32."""

import pytest
import torch

pytestmark = pytest.mark.gpu

SIGN = -2 ** 31


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def test_count_tokens(dev):
    from llmnputest_amd import ops
    b, v = 5, 20011
    g = torch.Generator(device="cuda").manual_seed(3)
    n = [0, 1, 4000, 77, 30000]
    cu = ints([0, 0, 1, 4001, 4078, 34078])
    tokens = (v * torch.rand(34078, device="cuda", generator=g) ** 4).to(torch.int32)
    tokens[::50] = -1
    tokens[7::50] = v
    tokens[9::50] = 2 ** 31 - 1
    counts = torch.randint(-5, 5, (b, v + 3), dtype=torch.int32, device="cuda", generator=g)[:, :v]
    want = torch.zeros((b, v), dtype=torch.int64, device="cuda")
    for i in range(b):
        t = tokens[int(cu[i]):int(cu[i + 1])].long()
        t = t[(t >= 0) & (t < v)]
        want[i] = torch.bincount(t, minlength=v)
    ops.count_tokens(counts, tokens, cu, start=True)
    assert torch.equal(counts.long(), want)
    ops.count_tokens(counts, tokens, cu)                       # added
    assert torch.equal(counts.long(), 2 * want)
    one = ints([0, v - 1, v, -1, 5])
    ops.count_tokens(counts, one)
    want *= 2
    for i, t in enumerate(one.tolist()):
        if 0 <= t < v:
            want[i, t] += 1
    assert torch.equal(counts.long(), want)
    ops.count_tokens(counts, tokens, cu, prompt=True)          # the sign bit, once
    ops.count_tokens(counts, one, prompt=True)
    has = torch.zeros((b, v), dtype=torch.bool, device="cuda")
    for i in range(b):
        t = tokens[int(cu[i]):int(cu[i + 1])].long()
        has[i, t[(t >= 0) & (t < v)]] = True
        if 0 <= int(one[i]) < v:
            has[i, int(one[i])] = True
    assert torch.equal(counts.long(), torch.where(has, want + SIGN, want))
    ops.count_tokens(counts, tokens[:0], ints([0] * (b + 1)), start=True)
    assert not bool(counts.any())


def reference(x, counts, r, p, f, bias, mask, rows):
    """The steps, each rounded to fp32, as the definition has them."""
    x = x.float()
    if counts is not None:
        n = counts & (2 ** 31 - 1)
        one = torch.ones(len(x), device="cuda")
        r, p, f = (one * d if t is None else t for t, d in ((r, 1), (p, 0), (f, 0)))
        hit = counts != 0
        y = torch.where(x > 0, x / r[:, None], x * r[:, None])
        y = y - f[:, None] * n
        y = torch.where(n > 0, y - p[:, None], y)
        x = torch.where(hit, y, x)
    if bias is not None:
        ids, values, cu = (t.tolist() for t in bias)
        v = torch.tensor(bias[1].tolist(), dtype=torch.float32)
        add = torch.zeros(x.shape, dtype=torch.float32)
        for i in range(len(x)):
            for k in range(cu[i], cu[i + 1]):
                if 0 <= ids[k] < x.shape[1]:
                    add[i, ids[k]] += v[k]
        x = x + add.cuda()
    if mask is not None:
        bits = (mask[:, :, None] >> torch.arange(32, device="cuda") & 1).flatten(1)[:, :x.shape[1]].bool()
        for i in range(len(x)):
            row = i if rows is None else int(rows[i])
            if row >= len(mask):
                x[i] = float("-inf")
            elif row >= 0:
                x[i] = x[i].masked_fill(~bits[row], float("-inf"))
    return x


CASES = [
    # b, v, bf16, penalties, biases, masks, rows
    (1, 1, False, True, 0, 0, False),
    (1, 100352, False, True, 0, 0, False),
    (3, 1000, False, False, 5, 0, False),
    (2, 4097, True, True, 40, 2, False),
    (5, 50001, False, True, 300, 3, True),
    (9, 248320, True, True, 0, 4, True),
    (64, 70001, False, True, 20, 7, True),
    (130, 33, True, True, 3, 130, False),
    (4, 8191, False, False, 0, 4, False),
]


@pytest.mark.parametrize("case", CASES, ids=[f"b{c[0]}v{c[1]}{'h' if c[2] else ''}" for c in CASES])
def test_adjust_logits(dev, case):
    from llmnputest_amd import ops
    b, v, half, pen, n_bias, n_mask, by_row = case
    g = torch.Generator(device="cuda").manual_seed(v)
    dt = torch.bfloat16 if half else torch.float32
    wide = (4 * torch.randn((b, v + 5), device="cuda", generator=g)).to(dt)
    x = wide[:, 3:v + 3]                       # rows that begin anywhere
    if v > 100:
        x[0, 50], x[-1, 60], x[0, 70] = float("inf"), float("-inf"), 0.0
    counts = r = p = f = bias = mask = rows = None
    if pen:
        counts = torch.randint(0, 40, (b, v), device="cuda", generator=g)
        counts = torch.where(counts < 4, counts, torch.where(counts < 7, SIGN + counts - 4, 0)).to(torch.int32)
        r = 0.5 + torch.rand(b, device="cuda", generator=g)
        p, f = torch.randn(b, device="cuda", generator=g), torch.randn(b, device="cuda", generator=g)
    if n_bias:
        ids = torch.randint(-2, v + 2, (b * n_bias,), dtype=torch.int32, device="cuda", generator=g)
        ids[::3] = ids[0]                      # the same token again
        cut = sorted(int(t) for t in torch.randint(0, b * n_bias + 1, (b - 1,), device="cuda", generator=g))
        bias = (ids, torch.randn(b * n_bias, device="cuda", generator=g), ints([0, *cut, b * n_bias]))
    if n_mask:
        mask = torch.randint(-2 ** 31, 2 ** 31, (n_mask, (v + 31) // 32), device="cuda", generator=g).to(torch.int32)
        mask[-1] = 0                           # nothing allowed
        if by_row:
            rows = ints([(-1, n_mask, 0, n_mask - 1)[i] if i < 4 else i % n_mask for i in range(b)])
    want = reference(x, counts, r, p, f, bias, mask, rows)
    keys = torch.empty(b, dtype=torch.int64, device="cuda")
    before = x.clone()
    out, token = ops.adjust_logits(x, counts, r, p, f, bias, mask, rows, keys=keys)
    assert torch.equal(x, before)
    assert torch.equal(out, want.to(dt))
    best = torch.where(want.isnan(), float("inf"), want)
    first = torch.where(best == best.amax(-1, keepdim=True), torch.arange(v, device="cuda"), v).amin(-1)
    assert torch.equal(token.long(), first)
    assert torch.equal(keys & 0xFFFFFFFF, 0xFFFFFFFF - first)
    # in place, and again from the same workspace
    y, again = ops.adjust_logits(x, counts, r, p, f, bias, mask, rows, out=x)
    assert y is x and torch.equal(x, out) and torch.equal(again, token)
    rest = torch.cat((wide[:, :3], wide[:, v + 3:]), 1)
    assert not bool(rest.isinf().any())


def test_nan_is_greatest(dev):
    from llmnputest_amd import ops
    x = torch.randn((3, 5000), device="cuda")
    x[0, 4000], x[0, 4500] = float("nan"), float("nan")
    x[1, 10] = float("nan")
    mask = torch.full((3, 157), -1, dtype=torch.int32, device="cuda")
    mask[1, 0] = ~(1 << 10)                    # not allowed: -inf, no NaN
    out, token = ops.adjust_logits(x, mask=mask)
    assert int(token[0]) == 4000 and bool(out[0, 4000].isnan())
    assert out[1, 10] == float("-inf") and not bool(out[1].isnan().any())
    assert int(token[1]) == int(out[1].argmax()) and int(token[2]) == int(x[2].argmax())
