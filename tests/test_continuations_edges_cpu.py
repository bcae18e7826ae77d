"""Several continuations of a prompt without a GPU: what the kernels' sources have to say about memory that
waves share, and what the decoder and the rules do on the host."""

import subprocess
import sys
from pathlib import Path

from llmnputest_amd import _lib, ops
from llmnputest_amd.granite import GraniteConfig, GraniteDecoder, GraniteWeights

CSRC = Path(__file__).resolve().parents[1] / "llmnputest_amd" / "csrc"


def test_prefix_tiles_wait_for_the_first():
    """A prefix part's first tile of K is scored in front of the loop over the tiles, whose first step fetches the
    third tile into the same LDS: a barrier that every wave reaches lies between the two."""
    text = (CSRC / "attn_prefix.hip").read_text()
    between = text[text.index("m[n] = greatest(n, 0, 4);"):text.index("tile(t, std::true_type{}")]
    assert "\n  if (nt > 2) __syncthreads();\n" in between   # at the function's own depth, not under `busy`


def test_eviction_leaves_the_steps_workspace(monkeypatch):
    """The step's graphs hold the address of the decoder's workspace. With as many kv heads as query heads an
    eviction needs more than a step: it must not replace that memory."""
    lib = _lib.lib()
    assert lib.q4nx_kv_evict_ws_bytes(20, 40, 16448) > lib.q4nx_gqa_decode_weights_ws_bytes(20, 40, 40, 64, 16448)
    cfg = GraniteConfig(hidden=256, inter=256, n_layers=2, n_q=4, n_kv=4, vocab=256)
    dec = GraniteDecoder(GraniteWeights(cfg), max_batch=2, max_len=16448, device="cpu", track_weights=True)
    dec.ws = ops.Workspace(ops.WS_COUNTER_BYTES, device="cpu")
    held, calls = dec.ws.buf, []

    def kv_evict(k, v, w, lens, budget, recent, rope=None, into=None, max_len=None, ws=None):
        calls.append(lens.tolist())
        if ws is not None:
            ws.get(lib.q4nx_kv_evict_ws_bytes(k.shape[0], k.shape[1], k.shape[2]))

    monkeypatch.setattr(ops, "kv_evict", kv_evict)
    assert dec.evict([16400, 9], 100, 10) == [100, 9]
    assert calls == [[16400, 9]] * 2 and dec.ws.buf is held


def test_import_needs_no_private_names():
    """The package is imported also where torch's own name for the question whether a stream captures is gone."""
    code = "import torch; del torch._C._cuda_isCurrentStreamCapturing; import llmnputest_amd.ops"
    assert subprocess.run([sys.executable, "-c", code], cwd=CSRC.parents[1]).returncode == 0
