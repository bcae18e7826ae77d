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


def pools(dec):
    return [t.clone() for t in (dec.kv.pool, dec.kv.table, dec.kv.refs)]


@pytest.mark.parametrize("page", [32, 64])
def test_no_row_goes_into_a_shared_page(weights, page):
    """After a fork: positions in the shared prefix are refused by step(), generate() and capture(), with
    nothing written, whichever sequence they belong to; positions behind it are taken."""
    dec = decoder(weights, 3, page_len=page)
    dec.seed_cache(150, seed=6)
    dec.fork([0], [1], [140])
    full = 140 // page * page
    before = pools(dec)
    for bad in ([full - 1, 150, 150], [150, 0, 150], [0, 0, 150], [150, full - 1, 150]):
        with pytest.raises(ValueError, match="shares"):
            dec.step([1, 2, 3], bad)
        with pytest.raises(ValueError, match="shares"):
            dec.generate([1, 2, 3], bad, 40)
    with pytest.raises(ValueError, match="shares"):
        dec.step([1], [5])
    with pytest.raises(ValueError, match="shares"):
        dec.capture(3)               # its warm step would write at positions 0
    assert all(torch.equal(a, b) for a, b in zip(before, pools(dec)))
    dec.step([1, 2, 3], [full, 150, 0])
    dec.generate([1, 2, 3], [150, full, 17], 5)
    dec.step([1, 2, 3], [140, 140, 3])


def test_a_shared_page_is_ones_own_when_the_others_have_ended(weights):
    """The source may be wound back once both copies have other pages; a copy after reset(); what a fork
    from a fork shares is refused in all three."""
    dec = decoder(weights, 3)
    dec.seed_cache(150, seed=6)
    dec.fork([0], [1], [130])
    dec.fork([1], [2], [70])
    for bad in ([63, 200, 200], [200, 63, 200], [200, 200, 63], [64, 200, 200], [200, 127, 200]):
        with pytest.raises(ValueError, match="shares"):
            dec.step([1, 1, 1], bad)
    dec.step([1, 1, 1], [128, 128, 64])
    dec.reset([1])
    with pytest.raises(ValueError, match="shares"):
        dec.step([1, 1, 1], [63, 0, 200])
    dec.step([1, 1, 1], [64, 0, 64])          # the pages from 64 on were shared with sequence 1 alone
    with pytest.raises(ValueError, match="shares"):
        dec.generate([1, 1, 1], [60, 0, 200], 10)
    dec.fork([1], [2], [0])
    dec.step([1, 1, 1], [0, 0, 0])
    new = decoder(weights, 3)
    for d in (dec, new):
        d.seed_cache(64, seed=2)
    assert (dec.generate([5, 6, 7], [10, 64, 3], 9)[0] == new.generate([5, 6, 7], [10, 64, 3], 9)[0]).all()


def test_a_sequence_wound_back_is_as_new(weights):
    """A copy that was given up and its source, both started over: the logits of a decoder never forked."""
    dec, new = decoder(weights, 2, 128), decoder(weights, 2, 128)
    dec.seed_cache(100, seed=6)
    dec.fork([0], [1], [100])
    dec.reset([0, 1])
    for i in range(3):
        assert torch.equal(dec.step([9 + i, 3], [i, i]), new.step([9 + i, 3], [i, i]))


def test_nothing_stays_shared_after_a_fork_that_failed(weights):
    """One of two pairs cannot be done: the other's pages are not left shared without a guard."""
    dec = decoder(weights, 4)
    dec.seed_cache(150, seed=6)
    dec.kv.free([2])
    with pytest.raises(RuntimeError, match="prefix"):
        dec.fork([0, 2], [1, 3], [130, 130])
    refs, table = dec.kv.refs.cpu(), dec.kv.table.cpu()
    assert int(refs.max()) == 1 and (table >= 0).all() and int(refs.sum()) == table.numel()
    dec.step([1, 2, 3, 4], [0, 0, 0, 0])
