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
