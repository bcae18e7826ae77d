"""Rules for the tokens of a batch of sequences: penalties for what was said, biases, and masks of allowed
tokens, kept on the device and applied to each step's logits (`ops.adjust_logits`). No reference
counterpart: its tokens are chosen by transformers' generate (chat.py:74-78).

    rules = TokenRules(n_seqs=4, vocab=100352, repetition=1.1, frequency=[0.0, 0.2, 0.2, 0.5], max_biases=64)
    rules.begin([prompt_ids] * 4)                          # the prompts' tokens are seen, nothing is generated
    rules.set_bias([{50: -100.0}, {}, {}, {7: 2.5}])
    rules.allow(2, [3, 5, 8])                              # sequence 2 may say these
    dec = GraniteDecoder(w, max_batch=4, rules=rules)      # its greedy loop goes by them

Memory is laid out once, so that captured graphs see what is set later.
"""

from __future__ import annotations

import numpy as np
import torch

from . import ops


class TokenRules:
    """`counts` int32 [n_seqs, vocab] (`ops.count_tokens`), `repetition`, `presence`, `frequency` fp32
    [n_seqs]; `mask` int32 [rows, (vocab + 31) // 32] with `mask_rows` int32 [n_seqs], the row that a
    sequence goes by (-1: all allowed); at most max_biases biases in all, lists of up to hundreds a sequence
    (of 1 x 100352 logits, 10 us without: 300 neighbouring tokens 26 us, 4096 88, all 331).

    masks: a table of masks, int32 [rows, words], that sequences go by as `mask_rows` says (a grammar's
    states, say); without it every sequence has a row of its own, which `allow` sets."""

    def __init__(self, n_seqs: int, vocab: int, repetition=1.0, presence=0.0, frequency=0.0,
                 max_biases: int = 0, masks: torch.Tensor | None = None, device="cuda"):
        if n_seqs < 1 or vocab < 1 or max_biases < 0:
            raise ValueError("n_seqs and vocab must be positive, max_biases not negative")
        dev = self.device = torch.device(device)
        self.n_seqs, self.vocab, self.max_biases = n_seqs, vocab, max_biases
        words = (vocab + 31) // 32
        if masks is not None and (masks.dtype != torch.int32 or masks.dim() != 2 or masks.shape[1] != words
                                  or masks.shape[0] == 0):
            raise ValueError(f"masks must be int32 [rows, {words}]")
        self.counts = torch.zeros((n_seqs, vocab), dtype=torch.int32, device=dev)
        self.repetition, self.presence, self.frequency = (
            self._each(x, name) for x, name in ((repetition, "repetition"), (presence, "presence"),
                                                (frequency, "frequency")))
        if not bool((self.repetition > 0).all()):
            raise ValueError("repetition must be positive")
        self._shared = masks is not None
        self.mask = (masks.to(dev).contiguous() if self._shared
                     else torch.full((n_seqs, words), -1, dtype=torch.int32, device=dev))
        self.mask_rows = torch.full((n_seqs,), -1, dtype=torch.int32, device=dev)
        self.bias_ids = torch.zeros(max_biases, dtype=torch.int32, device=dev)
        self.bias_values = torch.zeros(max_biases, dtype=torch.float32, device=dev)
        self.bias_cu = torch.zeros(n_seqs + 1, dtype=torch.int32, device=dev)

    def _each(self, x, name: str) -> torch.Tensor:
        t = torch.as_tensor(x, dtype=torch.float32).to(self.device)
        if t.dim() == 0:
            t = t.repeat(self.n_seqs)
        if t.shape != (self.n_seqs,):
            raise ValueError(f"{name} must be one value or {self.n_seqs}")
        return t.contiguous().clone()

    def _lists(self, lists):
        if len(lists) != self.n_seqs:
            raise ValueError(f"a list for each of {self.n_seqs} sequences")
        flat = np.concatenate([np.asarray(x, dtype=np.int64).reshape(-1) for x in lists])
        if flat.size and (flat.min() < 0 or flat.max() >= self.vocab):
            raise ValueError(f"tokens must be in [0, {self.vocab})")
        cu = np.concatenate(([0], np.cumsum([len(x) for x in lists])))
        return (torch.from_numpy(flat.astype(np.int32)).to(self.device),
                torch.from_numpy(cu.astype(np.int32)).to(self.device))

    def begin(self, prompts) -> None:
        """Nothing is generated yet; the tokens of prompts (a list per sequence) are seen."""
        tokens, cu = self._lists(prompts)
        ops.count_tokens(self.counts, tokens, cu, prompt=True, start=True)

    def count(self, tokens: torch.Tensor) -> None:
        """One generated token of each of the first len(tokens) sequences (int32, on the device)."""
        ops.count_tokens(self.counts[:tokens.numel()], tokens)

    def set_bias(self, biases) -> None:
        """A dict of token: value per sequence, in place of what was set."""
        ids, cu = self._lists([list(x) for x in biases])
        n = ids.numel()
        if n > self.max_biases:
            raise ValueError(f"{n} biases, max_biases is {self.max_biases}")
        self.bias_ids[:n] = ids
        self.bias_values[:n] = torch.tensor([float(v) for x in biases for v in x.values()], dtype=torch.float32,
                                            device=self.device)
        self.bias_cu.copy_(cu)

    def allow(self, seq: int, tokens=None) -> None:
        """Sequence seq may say these tokens alone (None: all)."""
        if self._shared:
            raise ValueError("the masks are a table: set mask_rows")
        if not 0 <= seq < self.n_seqs:
            raise ValueError(f"sequences must be in [0, {self.n_seqs})")
        if tokens is None:
            self.mask_rows[seq] = -1
            return
        t = np.asarray(tokens, dtype=np.int64).reshape(-1)
        if t.size and (t.min() < 0 or t.max() >= self.vocab):
            raise ValueError(f"tokens must be in [0, {self.vocab})")
        words = np.zeros(self.mask.shape[1], np.uint32)
        np.bitwise_or.at(words, t // 32, np.uint32(1) << (t % 32).astype(np.uint32))
        self.mask[seq].copy_(torch.from_numpy(words.view(np.int32)))
        self.mask_rows[seq] = seq

    def apply(self, logits: torch.Tensor, out: torch.Tensor | None = None, tokens: torch.Tensor | None = None,
              keys: torch.Tensor | None = None, ws: ops.Workspace | None = None):
        """The rules on logits [b, vocab] of the first b sequences: (out, tokens) as
        `ops.adjust_logits` gives them."""
        b = logits.shape[0]
        if b > self.n_seqs:
            raise ValueError(f"logits of {b} sequences, the rules have {self.n_seqs}")
        bias = (self.bias_ids, self.bias_values, self.bias_cu[:b + 1]) if self.max_biases else None
        return ops.adjust_logits(logits, self.counts[:b], self.repetition[:b], self.presence[:b],
                                 self.frequency[:b], bias=bias, mask=self.mask, mask_rows=self.mask_rows[:b],
                                 out=out, tokens=tokens, keys=keys, ws=ws)
