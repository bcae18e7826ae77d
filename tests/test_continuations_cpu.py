"""The calls for several continuations of a prompt without a GPU: their workspaces' sizes, and arguments
that are refused before any launch."""

import ctypes as C

import pytest
import torch

from llmnputest_amd import _lib, ops
from llmnputest_amd.rules import TokenRules

ERR_ARG, ERR_SHAPE, ERR_WS = -1, -2, -3
AT = 0x10000   # aligned, never read: validation fails first
BIG = 1 << 40


def refused(name, args, **change):
    a = dict(args)
    assert set(change) <= set(a), set(change) - set(a)
    a.update(change)
    rc = getattr(_lib.lib(), name)(*a.values())
    return rc, _lib.lib().q4nx_last_error().decode()


PREFIX = dict(q=AT, kp=AT, vp=AT, ps=8 * 100 * 64, ph=100 * 64, plens=AT, cu=AT, p=2, most_p=100, k=AT, v=AT,
              bs=8 * 50 * 64, hs=50 * 64, lens=AT, most=50, out=AT, of=None, b=4, hq=40, hkv=8, d=64, scale=0.1,
              ws=AT, wn=BIG, stream=None)
WEIGHTS = dict(q=AT, k=AT, v=AT, bs=8 * 50 * 64, hs=50 * 64, lens=AT, most=50, w=AT, wb=8 * 50, wh=50, start=0, out=AT,
               of=None, b=4, hq=40, hkv=8, d=64, scale=0.1, ws=AT, wn=BIG, stream=None)
EVICT = dict(k=AT, v=AT, bs=8 * 50 * 64, hs=50 * 64, w=AT, wb=8 * 50, wh=50, lens=AT, most=50, budget=20, recent=5,
             tab=AT, max_pos=50, k2=2 * AT, v2=2 * AT, obs=8 * 20 * 64, ohs=20 * 64, w2=2 * AT, owb=8 * 20, owh=20,
             room=20, lens2=AT, kept=AT, b=4, hkv=8, d=64, ws=AT, wn=BIG, stream=None)
COUNT = dict(counts=AT, stride=100, vocab=100, b=4, tokens=AT, n=9, cu=AT, prompt=0, start=0, stream=None)
LOGITS = dict(x=AT, bf16=0, stride=100, out=AT, os=100, vocab=100, b=4, counts=AT, cs=100, rep=AT, pres=AT, freq=AT,
              ids=AT, values=AT, n=3, cu=AT, mask=AT, ms=4, n_mask=2, rows=AT, tokens=AT, keys=AT, ws=AT, wn=BIG,
              stream=None)


@pytest.mark.parametrize("change,code", [
    (dict(q=None), ERR_ARG), (dict(lens=None), ERR_ARG), (dict(out=None), ERR_ARG), (dict(kp=None), ERR_ARG),
    (dict(v=None), ERR_ARG), (dict(plens=None), ERR_ARG), (dict(cu=None), ERR_ARG), (dict(q=AT + 8), ERR_ARG),
    (dict(k=AT + 8), ERR_ARG), (dict(vp=AT + 2), ERR_ARG), (dict(out=AT + 4), ERR_ARG), (dict(of=AT + 8), ERR_ARG),
    (dict(scale=-0.1), ERR_ARG), (dict(scale=float("nan")), ERR_ARG), (dict(b=0), ERR_SHAPE), (dict(hq=41), ERR_SHAPE),
    (dict(hq=136), ERR_SHAPE), (dict(hkv=0), ERR_SHAPE), (dict(d=96), ERR_SHAPE), (dict(p=(1 << 20) + 1), ERR_SHAPE),
    (dict(p=-1), ERR_SHAPE), (dict(most_p=-1), ERR_SHAPE), (dict(most=1 << 24), ERR_SHAPE), (dict(most=51), ERR_SHAPE),
    (dict(most_p=101), ERR_SHAPE), (dict(hs=50 * 64 + 4), ERR_SHAPE), (dict(bs=50 * 64), ERR_SHAPE),
    (dict(ps=100 * 64), ERR_SHAPE), (dict(ws=None), ERR_WS), (dict(wn=1000), ERR_WS), (dict(ws=AT + 16), ERR_WS)])
def test_prefix_refusals(change, code):
    rc, msg = refused("q4nx_gqa_prefix_decode", PREFIX, **change)
    assert rc == code and msg.startswith("q4nx_gqa_prefix_decode"), msg


@pytest.mark.parametrize("change,code", [
    (dict(q=None), ERR_ARG), (dict(w=None), ERR_ARG), (dict(out=None), ERR_ARG), (dict(k=AT + 8), ERR_ARG),
    (dict(out=AT + 4), ERR_ARG), (dict(scale=-1.0), ERR_ARG), (dict(hq=7), ERR_SHAPE), (dict(d=32), ERR_SHAPE),
    (dict(most=0), ERR_SHAPE), (dict(most=51), ERR_SHAPE), (dict(wh=49), ERR_SHAPE), (dict(wb=8 * 49), ERR_SHAPE),
    (dict(hs=50 * 64 + 2), ERR_SHAPE), (dict(ws=None), ERR_WS), (dict(wn=65535), ERR_WS)])
def test_weights_refusals(change, code):
    rc, msg = refused("q4nx_gqa_decode_weights", WEIGHTS, **change)
    assert rc == code and msg.startswith("q4nx_gqa_decode_weights"), msg


@pytest.mark.parametrize("change,code", [
    (dict(k=None), ERR_ARG), (dict(w=None), ERR_ARG), (dict(kept=None), ERR_ARG), (dict(lens2=None), ERR_ARG),
    (dict(k=AT + 8), ERR_ARG), (dict(tab=AT + 4), ERR_ARG), (dict(k2=AT), ERR_ARG), (dict(v2=AT), ERR_ARG),
    (dict(w2=AT), ERR_ARG), (dict(k2=AT, v2=AT, w2=AT), ERR_ARG),      # in place, other strides
    (dict(budget=0), ERR_SHAPE), (dict(recent=21), ERR_SHAPE), (dict(recent=-1), ERR_SHAPE), (dict(d=80), ERR_SHAPE),
    (dict(most=0), ERR_SHAPE), (dict(most=51), ERR_SHAPE), (dict(room=19), ERR_SHAPE), (dict(owh=19), ERR_SHAPE),
    (dict(ohs=19 * 64), ERR_SHAPE), (dict(max_pos=49), ERR_SHAPE), (dict(wh=40), ERR_SHAPE), (dict(ws=None), ERR_WS),
    (dict(wn=65536), ERR_WS)])
def test_evict_refusals(change, code):
    rc, msg = refused("q4nx_kv_evict", EVICT, **change)
    assert rc == code and msg.startswith("q4nx_kv_evict"), msg


@pytest.mark.parametrize("change,code", [
    (dict(counts=None), ERR_ARG), (dict(tokens=None), ERR_ARG), (dict(vocab=0), ERR_SHAPE), (dict(b=0), ERR_SHAPE),
    (dict(b=65536), ERR_SHAPE), (dict(n=-1), ERR_SHAPE), (dict(stride=99), ERR_SHAPE), (dict(cu=None), ERR_SHAPE)])
def test_count_refusals(change, code):
    rc, msg = refused("q4nx_count_tokens", COUNT, **change)
    assert rc == code and msg.startswith("q4nx_count_tokens"), msg


@pytest.mark.parametrize("change,code", [
    (dict(x=None), ERR_ARG), (dict(out=None), ERR_ARG), (dict(counts=None), ERR_ARG), (dict(ids=None), ERR_ARG),
    (dict(values=None), ERR_ARG), (dict(cu=None), ERR_ARG), (dict(n=-1), ERR_ARG), (dict(vocab=0), ERR_SHAPE),
    (dict(b=4097), ERR_SHAPE), (dict(stride=99), ERR_SHAPE), (dict(os=99), ERR_SHAPE), (dict(cs=99), ERR_SHAPE),
    (dict(ms=3), ERR_SHAPE), (dict(n_mask=0), ERR_SHAPE), (dict(rows=None), ERR_SHAPE), (dict(mask=None), ERR_SHAPE),
    (dict(ws=None), ERR_WS), (dict(wn=65535), ERR_WS), (dict(ws=AT + 8), ERR_WS)])
def test_logits_refusals(change, code):
    rc, msg = refused("q4nx_adjust_logits", LOGITS, **change)
    assert rc == code and msg.startswith("q4nx_adjust_logits"), msg


def test_workspaces():
    lib = _lib.lib()
    size = lib.q4nx_gqa_prefix_decode_ws_bytes
    assert size(4, 40, 8, 64, 2, 1000, 500) >= 65536 + 4 * 40 * 2 * 68 * 4      # a part of each kind
    assert size(4, 40, 8, 64, 0, 0, 0) == 65536 and size(1, 8, 8, 128, 1, 512, 0) == 65536   # one launch
    for bad in ((0, 40, 8, 64, 1, 1, 1), (4, 40, 7, 64, 1, 1, 1), (4, 40, 8, 65, 1, 1, 1), (4, 40, 8, 64, -1, 1, 1)):
        assert size(*bad) == 0
    size = lib.q4nx_gqa_decode_weights_ws_bytes
    # scores of the longest length, and records
    assert size(8, 40, 8, 64, 32768) >= 65536 + 8 * 40 * (32768 + 68) * 4
    assert size(8, 40, 8, 64, 0) == 0
    assert lib.q4nx_kv_evict_ws_bytes(8, 8, 4096) >= 65536 + 64 * 4 and lib.q4nx_kv_evict_ws_bytes(0, 8, 9) == 0
    assert lib.q4nx_kv_evict_ws_bytes(8, 8, 40000) >= 65536 + 64 * 40000 * 4


def test_more_parts_than_a_wave_has_lanes_never():
    """A wave's lanes hold a (sequence, head)'s records: 32 parts of a prefix and 32 of an own cache."""
    lib = _lib.lib()
    for b in (1, 2, 3, 16, 64, 200):
        for most in (1025, 5000, 70000, (1 << 24) - 1):
            n = (lib.q4nx_gqa_prefix_decode_ws_bytes(b, 8, 4, 64, 1, most, most) - 65536) // (b * 8 * 68 * 4)
            assert 2 <= n <= 64
            one = lib.q4nx_gqa_prefix_decode_ws_bytes(b, 8, 4, 64, 0, 0, most) - 65536
            assert one // (b * 8 * 68 * 4) <= 32


def test_host_checks():
    """What the wrappers refuse whatever the device."""
    q = torch.zeros((2, 4, 64), dtype=torch.bfloat16)
    with pytest.raises((ValueError, RuntimeError, AssertionError)):   # no GPU: not on the current device
        ops.gqa_prefix_decode(q, q, q, q, q, q, q)
    with pytest.raises(ValueError, match="positive"):
        TokenRules(0, 10, device="cpu")
    with pytest.raises(ValueError, match="repetition"):
        TokenRules(2, 10, repetition=0.0, device="cpu")
    with pytest.raises(ValueError, match="one value or 2"):
        TokenRules(2, 10, presence=[1.0, 2.0, 3.0], device="cpu")
    with pytest.raises(ValueError, match="masks"):
        TokenRules(2, 100, masks=torch.zeros((3, 3), dtype=torch.int32), device="cpu")


def test_rules_on_the_host():
    r = TokenRules(3, 70, max_biases=3, device="cpu")
    r.set_bias([{5: 1.5}, {}, {69: -2.0, 0: 3.0}])
    assert r.bias_ids.tolist() == [5, 69, 0] and r.bias_values.tolist() == [1.5, -2.0, 3.0]
    assert r.bias_cu.tolist() == [0, 1, 1, 3]
    r.set_bias([{}, {7: 4.0}, {}])
    assert r.bias_cu.tolist() == [0, 0, 1, 1] and int(r.bias_ids[0]) == 7
    for bad in ([{}, {}], [{70: 1.0}, {}, {}], [{-1: 1.0}, {}, {}], [{1: 0, 2: 0}, {1: 0, 2: 0}, {}]):
        with pytest.raises(ValueError):
            r.set_bias(bad)
    r.allow(1, [0, 31, 32, 69])
    bits = [(int(r.mask[1, t // 32]) >> (t % 32)) & 1 for t in range(70)]
    assert [t for t in range(70) if bits[t]] == [0, 31, 32, 69] and r.mask_rows.tolist() == [-1, 1, -1]
    r.allow(1)
    assert r.mask_rows.tolist() == [-1, -1, -1]
    r.allow(0, [])
    assert not bool(r.mask[0].any()) and r.mask_rows.tolist() == [0, -1, -1]
    for bad in ((3, [1]), (0, [70]), (0, [-1])):
        with pytest.raises(ValueError):
            r.allow(*bad)
    with pytest.raises(ValueError, match="table"):
        TokenRules(2, 64, masks=torch.zeros((5, 2), dtype=torch.int32), device="cpu").allow(0, [1])
