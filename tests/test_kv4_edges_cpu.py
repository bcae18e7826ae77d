"""Calls of the 4-bit K/V cache's C entry points that were refused for nothing, without a GPU: they get as
far as the workspace, which they are not given."""

import pytest

from llmnputest_amd import _lib
from tests.test_kv4_cpu import ERR_WS, P, attn, cache


@pytest.mark.parametrize("new", [1 << 20, (1 << 20) + 1, 1 << 24, 2 ** 31 - 1])
def test_blocks_of_many_tokens_are_taken(new):
    """More than 2^20 tokens of one sequence: the rows in all are what is bounded (below 2^30 with heads)."""
    size = _lib.lib().q4nx_kv4_attn_ws_bytes(cache(), 8, 1 << 22, new, 1000, 0, 0)
    assert size == _lib.lib().q4nx_kv4_attn_ws_bytes(cache(), 8, 1 << 22, 1, 1000, 0, 0) > 0
    assert attn(cache(), cu=P, total=64, hq=8, new=new, split=2)[0] == ERR_WS
