"""GraniteDecoder with its K/V cache in 4-bit pages: every layer's appended rows and attention against
the numpy oracle on the bytes of the pool, the graph loop against single steps, selected pages, forks."""

import numpy as np
import pytest
import torch

from llmnputest_amd.granite import GraniteConfig, GraniteDecoder, GraniteWeights
from oracle import kv4_oracle as ko

pytestmark = pytest.mark.gpu

CFG = GraniteConfig(n_layers=2, vocab=4096)


@pytest.fixture(scope="module")
def weights():
    return GraniteWeights.synthetic(CFG, seed=3, device="cuda")


def decoder(weights, batch, max_len, **kw):
    return GraniteDecoder(weights, max_batch=batch, max_len=max_len, kv="q4", **kw)


@pytest.mark.parametrize("batch,page", [(1, 64), (3, 32)])
def test_layers_against_the_oracle(weights, batch, page):
    dec = decoder(weights, batch, 256, page_len=page)
    dec.seed_cache(100, seed=5)
    pos = [100, 37, 99][:batch]
    trace = []
    logits = dec.step([11, 222, 3333][:batch], pos, trace=trace)
    assert torch.isfinite(logits).all()
    table = dec.kv.table.cpu().numpy()
    for li, t in enumerate(trace):
        pages = ko.Pages(dec.kv.pool[li].cpu().numpy(), CFG.n_kv, 64, page)
        for b in range(batch):
            # the row that was appended: the quantised k and v of this step
            for h in range(CFG.n_kv):
                got = pages.values(table[b, pos[b] // page], h, pos[b] % page)
                for y, name in zip(got, ("k", "v")):
                    x = ko.bf16_f32(t[name][b, h])
                    codes, d, m = ko.quant(x)
                    want = codes.reshape(-1, 32) * ko.bf16_f32(d)[:, None].astype(np.float64) \
                        + ko.bf16_f32(m)[:, None]
                    assert np.array_equal(y, want.reshape(-1).astype(np.float32))
            q = ko.bf16_f32(t["q"][b]).astype(np.float64)[None]
            want, bound = ko.attention(pages, table[b], q, [pos[b] + 1], CFG.scale)
            off = np.abs(ko.bf16_f32(t["attn"][b]) - want[0])
            assert (off <= bound[0] + 2.0 ** -8 * (np.abs(want[0]) + bound[0])).all()


def test_bf16_and_q4_caches_hold_the_same_context(weights):
    """seed_cache fills both kinds of cache from the same rows: what q4 stands for is within half a
    step (and d's rounding, 15 d 2^-8 at the top) of the bf16 rows."""
    a = GraniteDecoder(weights, max_batch=2, max_len=128)
    b = decoder(weights, 2, 128)
    for d in (a, b):
        d.seed_cache(70, seed=9)
    zero, cu = torch.zeros(2, dtype=torch.int32, device="cuda"), torch.tensor([0, 70, 140], dtype=torch.int32,
                                                                             device="cuda")
    for li in range(2):
        for got, want in zip(b.kv.read(li, zero, cu, dtype=torch.float32), (a.k_cache[li], a.v_cache[li])):
            x = want[:, :, :70].transpose(1, 2).reshape(140, CFG.n_kv, 2, 32).float()
            step = (x.amax(-1, keepdim=True) - x.amin(-1, keepdim=True)) / 15
            assert ((got.reshape(x.shape) - x).abs() <= step * (0.5 + 2.0 ** -7 + 15 * 2.0 ** -8)).all()


@pytest.mark.parametrize("batch,sparse", [(1, 0), (2, 0), (2, 3)])
def test_generate_equals_steps(weights, batch, sparse):
    """The graph loop's greedy tokens are those of eager steps."""
    start, n = [150, 131][:batch], 20
    dec = decoder(weights, batch, 256, sparse_pages=sparse)
    dec.seed_cache(150, seed=2)
    got, _ = dec.generate([7, 8][:batch], start, n)
    dec.seed_cache(150, seed=2)
    tok, want = [7, 8][:batch], []
    for i in range(n):
        logits = dec.step(tok, [s + i for s in start])
        tok = logits.argmax(-1).tolist()
        want.append(tok)
    assert np.array_equal(got, np.array(want).T)


def test_all_pages_selected_is_dense(weights):
    """With as many pages as there are, the chosen ones are all: the logits' bits."""
    out = []
    for sparse in (0, 4):
        dec = decoder(weights, 2, 256, sparse_pages=sparse, attn_splits=1)
        dec.seed_cache(200, seed=4)
        out.append(dec.step([5, 6], [200, 120]).clone())
    assert torch.equal(*out)


def test_fork(weights):
    """Two copies of a sequence give its logits, bit for bit, and go their own ways without touching it;
    pages are shared until they end."""
    dec = decoder(weights, 3, 256, attn_splits=2)
    dec.seed_cache(150, seed=6)
    dec.fork([0, 0], [1, 2], [140, 140])
    refs = dec.kv.refs.cpu()
    assert (refs == 3).sum() == 140 // 64 and int(dec.kv.status) == 0
    a = dec.step([9, 9, 9], [140] * 3).clone()
    assert torch.equal(a[0], a[1]) and torch.equal(a[0], a[2])
    b = dec.step([1, 2, 3], [141] * 3).clone()
    assert not torch.equal(b[0], b[1])
    one = decoder(weights, 3, 256, attn_splits=2)
    one.seed_cache(150, seed=6)
    assert torch.equal(one.step([9, 9, 9], [140] * 3)[0], a[0])
    assert torch.equal(one.step([1, 2, 3], [141] * 3)[0], b[0])
    for bad in (([0], [0], [5]), ([0], [1, 2], [5]), ([0, 1], [2, 2], [5, 5]), ([0, 0], [1, 2], [5, 6]),
                ([3], [1], [5]), ([0], [1], [257])):
        with pytest.raises(ValueError):
            dec.fork(*bad)


def test_refusals(weights):
    with pytest.raises(ValueError, match="kv"):
        GraniteDecoder(weights, kv="q8")
    with pytest.raises(ValueError, match="sparse_pages"):
        GraniteDecoder(weights, sparse_pages=4)
    with pytest.raises(ValueError, match="fork"):
        GraniteDecoder(weights, max_batch=2, max_len=64).fork([0], [1], [3])
