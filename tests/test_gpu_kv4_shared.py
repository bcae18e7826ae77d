"""GraniteDecoder's sequences that share 4-bit pages: what a fork could not do is said, and no row is
written into a page that another sequence reads."""

import pytest
import torch

from llmnputest_amd.granite import GraniteConfig, GraniteDecoder, GraniteWeights

pytestmark = pytest.mark.gpu

CFG = GraniteConfig(n_layers=2, vocab=4096)


@pytest.fixture(scope="module")
def weights():
    return GraniteWeights.synthetic(CFG, seed=3, device="cuda")


def decoder(weights, batch, max_len=256, **kw):
    return GraniteDecoder(weights, max_batch=batch, max_len=max_len, kv="q4", attn_splits=2, **kw)


@pytest.mark.parametrize("length", [100, 128])
def test_a_fork_that_is_not_done_is_an_error(weights, length):
    """A source that has lost its pages: the pages that reserve() then finds do not hide it."""
    dec = decoder(weights, 3)
    dec.seed_cache(150, seed=6)
    dec.kv.free([0])
    with pytest.raises(RuntimeError, match="prefix"):
        dec.fork([0], [1], [length])


def test_seed_cache_after_a_fork(weights):
    """Every sequence gets the rows that a new decoder gives it, in pages of its own."""
    dec, new = decoder(weights, 3), decoder(weights, 3)
    dec.seed_cache(150, seed=6)
    dec.fork([0, 0], [1, 2], [140, 140])
    assert int(dec.kv.refs.max()) == 3
    for d in (dec, new):
        d.seed_cache(130, seed=8)
    assert int(dec.kv.refs.max()) == 1
    for li in range(CFG.n_layers):
        cu = torch.tensor([0, 130, 260, 390], dtype=torch.int32, device="cuda")
        for a, b in zip(*(d.kv.read(li, cu[:3] * 0, cu, total=390) for d in (dec, new))):
            assert torch.equal(a, b)
    assert torch.equal(dec.step([9, 8, 7], [130, 130, 64]), new.step([9, 8, 7], [130, 130, 64]))


def test_reset_gives_pages_of_ones_own(weights):
    dec = decoder(weights, 3)
    dec.seed_cache(150, seed=6)
    dec.fork([0, 0], [1, 2], [140, 140])
    dec.reset([1, 1])
    refs, table = dec.kv.refs.cpu(), dec.kv.table.cpu()
    assert (refs[table[0, :2].long()] == 2).all() and (refs[table[1].long()] == 1).all()
    assert (table >= 0).all() and int(refs.sum()) == table.numel()
    dec.reset([])
    for bad in ([3], [-1], [0, 7]):
        with pytest.raises(ValueError):
            dec.reset(bad)
    with pytest.raises(ValueError, match="reset"):
        GraniteDecoder(weights, max_batch=2, max_len=64).reset([0])
