"""Several continuations of a prompt without a GPU: what the kernels' sources have to say about memory that
waves share, and what the decoder and the rules do on the host."""

from pathlib import Path

CSRC = Path(__file__).resolve().parents[1] / "llmnputest_amd" / "csrc"


def test_prefix_tiles_wait_for_the_first():
    """A prefix part's first tile of K is scored in front of the loop over the tiles, whose first step fetches the
    third tile into the same LDS: a barrier that every wave reaches lies between the two."""
    text = (CSRC / "attn_prefix.hip").read_text()
    between = text[text.index("m[n] = greatest(n, 0, 4);"):text.index("tile(t, std::true_type{}")]
    assert "\n  if (nt > 2) __syncthreads();\n" in between   # at the function's own depth, not under `busy`
