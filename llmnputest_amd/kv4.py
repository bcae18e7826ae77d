"""A paged 4-bit K/V cache on the GPU: quantising writes, attention over it (single tokens and prompt
blocks), attention over the pages that a cheap score selects, and the pages' bookkeeping (reserve,
fork, free, compact). The format and every rule stand in include/q4nx_hip.h; all arithmetic runs in
libq4nx_hip.so. No reference counterpart: its cache is one dense bf16 buffer per sequence
(designs/granite_gemv/granite_attention.h:28-34).

    cache = Kv4Cache(n_layers=40, n_pages=2048, n_seqs=8, max_len=8192)
    cache.reserve([n + 128 for n in prompt_lens])           # pages for the prompts and what follows
    cache.append(layer, k, v, pos, cu, max_new=longest)     # k, v bf16 [rows, Hkv, D]
    out = cache.attn(layer, q, lens, cu=cu, max_new=longest)  # the prompt block, causal
    out = cache.attn(layer, q, lens)                        # one token per sequence
    sel = cache.select(layer, q, lens, n_sel=64)            # the 64 pages that matter most
    out = cache.attn(layer, q, lens, sel=sel)

As with the other ops, tensors must live on the current device and work goes to the current stream.
"""

from __future__ import annotations

import ctypes as C

import torch

from . import _lib, ops


def page_bytes(page_len: int = 64, n_kv_heads: int = 8, head_dim: int = 64) -> int:
    """Bytes of one page of one layer."""
    n = int(_lib.lib().q4nx_kv4_page_bytes(page_len, n_kv_heads, head_dim))
    if n == 0:
        raise ValueError(f"no pages of {page_len} positions (32, 64, 128), {n_kv_heads} kv heads "
                         f"(1..1024) of {head_dim} (64, 128)")
    return n


def _row_stride(table: torch.Tensor) -> int:
    """Entries from row to row of a page table; a single row's stride says nothing. Rows that overlap
    (an expanded row) keep their stride, which the library refuses."""
    return table.stride(0) if table.shape[0] > 1 else table.shape[1]


def _strides(t: torch.Tensor) -> tuple:
    """Strides, 0 where a dimension has one entry and its stride says nothing."""
    return tuple(x if n > 1 else 0 for n, x in zip(t.shape, t.stride()))


class Kv4Cache:
    """Pages of every layer (`pool` uint8 [n_layers, n_pages, page bytes]), the sequences' page table
    (`table` int32 [n_seqs, table_len], -1: none), their lengths (`lens` int32 [n_seqs]) and how many
    entries name each page (`refs` int32 [n_pages]). `status` (int32 [1]) is what the last
    bookkeeping call could not do. Writing and attention take lengths and positions from the caller;
    `lens` is theirs by default and what fork() and free() keep."""

    def __init__(self, n_layers: int, n_pages: int, n_seqs: int, max_len: int, n_kv_heads: int = 8,
                 head_dim: int = 64, page_len: int = 64, device="cuda"):
        if min(n_layers, n_pages, n_seqs, max_len) < 1:
            raise ValueError("n_layers, n_pages, n_seqs and max_len must be positive")
        dev = torch.device(device)
        size = page_bytes(page_len, n_kv_heads, head_dim)
        self._init(torch.zeros((n_layers, n_pages, size), dtype=torch.uint8, device=dev),
                   torch.full((n_seqs, -(-max_len // page_len)), -1, dtype=torch.int32, device=dev),
                   torch.zeros(n_seqs, dtype=torch.int32, device=dev),
                   torch.zeros(n_pages, dtype=torch.int32, device=dev), n_kv_heads, head_dim, page_len)

    @classmethod
    def over(cls, pool: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, refs: torch.Tensor, *,
             n_kv_heads: int = 8, head_dim: int = 64, page_len: int = 64) -> "Kv4Cache":
        """A cache over memory that the caller has."""
        c = cls.__new__(cls)
        c._init(pool, table, lens, refs, n_kv_heads, head_dim, page_len)
        return c

    def _init(self, pool, table, lens, refs, n_kv_heads, head_dim, page_len):
        size = page_bytes(page_len, n_kv_heads, head_dim)
        for t, name, dt, dim in ((pool, "pool", torch.uint8, 3), (table, "table", torch.int32, 2),
                                 (lens, "lens", torch.int32, 1), (refs, "refs", torch.int32, 1)):
            if not t.is_cuda or t.device != pool.device:
                raise ValueError(f"{name} must be on the pool's GPU, got {t.device}")
            if t.dtype != dt or t.dim() != dim or t.numel() == 0 or t.stride(-1) != 1:
                raise ValueError(f"{name} must be {dt} of {dim} dimensions, rows contiguous")
        if pool.shape[2] != size:
            raise ValueError(f"pool holds pages of {pool.shape[2]} bytes, expected {size}")
        if lens.shape[0] != table.shape[0] or refs.shape[0] != pool.shape[1]:
            raise ValueError("lens has an entry per sequence, refs one per page")
        self.pool, self.table, self.lens, self.refs = pool, table, lens, refs
        self.n_layers, self.n_pages, _ = pool.shape
        self.n_seqs, self.table_len = table.shape
        self.n_kv_heads, self.head_dim, self.page_len = n_kv_heads, head_dim, page_len
        self.max_len = self.table_len * page_len
        self.device = pool.device
        self._index = pool.get_device()
        self._lib = _lib.lib()
        self.status = torch.zeros(1, dtype=torch.int32, device=pool.device)
        self._layers = [_lib.Kv4(pool.data_ptr() + i * pool.stride(0), pool.stride(1), table.data_ptr(),
                                 _row_stride(table), self.n_pages, page_len, n_kv_heads, head_dim,
                                 self.n_seqs, self.table_len) for i in range(self.n_layers)]
        self._needs: dict = {}   # workspace bytes by the sizes that set them

    # ------------------------------------------------------------ arguments
    def _layer(self, layer: int, table: torch.Tensor | None):
        """The C view of a layer, and its sequences: those of `table` when one is given."""
        if not 0 <= layer < self.n_layers:
            raise IndexError(f"layer {layer} of {self.n_layers}")
        if self._index != torch.cuda.current_device():
            raise ValueError(f"the cache is on {self.device}, the current device is "
                             f"cuda:{torch.cuda.current_device()}")
        c = self._layers[layer]
        if table is None:
            return c, self.n_seqs
        self._tensor(table, "table", torch.int32)
        if table.dim() != 2 or table.stride(1) != 1 or table.numel() == 0:
            raise ValueError("table must be [sequences, pages], rows contiguous")
        v = _lib.Kv4.from_buffer_copy(c)
        v.table, v.table_stride = table.data_ptr(), _row_stride(table)
        v.n_seqs, v.table_len = table.shape
        return v, v.n_seqs

    def _tensor(self, t: torch.Tensor, name: str, dtype) -> None:
        if t.get_device() != self._index:
            raise ValueError(f"{name} must be on {self.device}, got {t.device}")
        if t.dtype != dtype:
            raise TypeError(f"{name} must be {dtype}, got {t.dtype}")

    def _ints(self, t: torch.Tensor, name: str, n: int) -> int:
        if t.get_device() != self._index or t.dtype != torch.int32:
            self._tensor(t, name, torch.int32)
        if t.shape != (n,) or not t.is_contiguous():
            raise ValueError(f"{name} must be {n} contiguous values")
        return t.data_ptr()

    def _call(self, name: str, *args) -> None:
        rc = getattr(self._lib, name)(*args)
        if rc:
            _lib.check(rc)

    def _list(self, x, name: str) -> torch.Tensor:
        t = torch.as_tensor(x, dtype=torch.int32, device=self.device) if not torch.is_tensor(x) else x
        self._tensor(t, name, torch.int32)
        if t.dim() != 1 or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous list")
        return t

    def _rows(self, k: torch.Tensor, v: torch.Tensor) -> tuple[int, int, int]:
        """Rows of k and v, their row and head strides."""
        for t, name in ((k, "k"), (v, "v")):
            if t.get_device() != self._index or t.dtype != torch.bfloat16:
                self._tensor(t, name, torch.bfloat16)
        shape, stride = k.shape, k.stride()
        if len(shape) != 3 or shape[1] != self.n_kv_heads or shape[2] != self.head_dim or stride[2] != 1:
            raise ValueError(f"k must be [rows, {self.n_kv_heads}, {self.head_dim}], channels contiguous")
        if v.shape != shape or (v.stride() != stride and _strides(v) != _strides(k)):
            raise ValueError("k and v must have one shape and one layout")
        return shape[0], stride[0] if shape[0] > 1 else 0, stride[1] if shape[1] > 1 else 0

    def _query(self, q: torch.Tensor) -> tuple[int, int, int]:
        """Rows, heads and row stride of q."""
        if q.get_device() != self._index or q.dtype != torch.bfloat16:
            self._tensor(q, "q", torch.bfloat16)
        shape, stride = q.shape, q.stride()
        if len(shape) != 3 or shape[2] != self.head_dim or stride[2] != 1 \
                or (shape[1] > 1 and stride[1] != self.head_dim):
            raise ValueError(f"q must be [rows, Hq, {self.head_dim}], heads contiguous")
        # a single row's stride says nothing
        return shape[0], shape[1], stride[0] if shape[0] > 1 else shape[1] * self.head_dim

    def _most(self, c, max_len: int | None) -> int:
        """The positions a sequence may have in a call."""
        cap = c.table_len * self.page_len
        return cap if max_len is None else min(cap, max_len)

    def _need(self, c, fn: str, *args) -> int:
        key = (fn, c.n_seqs, c.table_len, *args)
        n = self._needs.get(key)
        if n is None:
            if len(self._needs) > 4096:   # lengths that change from call to call
                self._needs.clear()
            n = self._needs[key] = int(getattr(_lib.lib(), fn)(c, *args))
        return n

    # ------------------------------------------------------------ rows
    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, pos: torch.Tensor,
               cu: torch.Tensor | None = None, max_new: int | None = None,
               table: torch.Tensor | None = None) -> None:
        """Writes rows k, v (bf16 [rows, Hkv, D], any row and head strides that are multiples of 8) at
        positions pos[b], pos[b] + 1, .. of every sequence: one row each, or rows cu[b] .. cu[b+1] - 1
        (int32 [n_seqs + 1]); max_new: at least the most rows of one sequence (default: all rows)."""
        c, b = self._layer(layer, table)
        n, row, head = self._rows(k, v)
        if cu is None and n != b:
            raise ValueError(f"{n} rows for {b} sequences (give cu for other numbers of rows)")
        if n == 0:
            return
        self._call_append(c, k, v, 0, n, row, head, 0, pos, cu, max_new or n)

    def append_cached(self, layer: int, k_cache: torch.Tensor, v_cache: torch.Tensor, pos: torch.Tensor,
                      cu: torch.Tensor | None = None, max_new: int | None = None,
                      table: torch.Tensor | None = None) -> None:
        """append() of rows that lie at their positions in a dense cache, bf16 [n_seqs, Hkv, L, D] as
        `ops.qkv_rope` writes it: positions pos[b] (and as many behind it as cu says)."""
        c, b = self._layer(layer, table)
        for t, name in ((k_cache, "k_cache"), (v_cache, "v_cache")):
            self._tensor(t, name, torch.bfloat16)
            if t.dim() != 4 or t.shape[0] < b or t.shape[1] != self.n_kv_heads \
                    or t.shape[3] != self.head_dim or t.stride(3) != 1 or t.numel() == 0:
                raise ValueError(f"{name} must be [{b}, {self.n_kv_heads}, L, {self.head_dim}]")
        seq, head, row, _ = strides = _strides(k_cache)
        if k_cache.shape != v_cache.shape or _strides(v_cache) != strides:
            raise ValueError("k_cache and v_cache must have one shape and one layout")
        n = k_cache.shape[2]
        self._call_append(c, k_cache, v_cache, 1, n, row, head, seq, pos, cu, max_new or n)

    def _call_append(self, c, k, v, by_position, rows, row, head, seq, pos, cu, max_new):
        self._call("q4nx_kv4_append", c, k.data_ptr(), v.data_ptr(), by_position, rows, row, head, seq,
                  self._ints(pos, "pos", c.n_seqs),
                  None if cu is None else self._ints(cu, "cu", c.n_seqs + 1),
                  1 if cu is None else max_new, ops._stream())

    def read(self, layer: int, pos: torch.Tensor, cu: torch.Tensor | None = None,
             total: int | None = None, max_new: int | None = None, dtype=torch.bfloat16,
             table: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """What the cache holds at those positions, k and v [total, Hkv, D] (bf16 or fp32). total: the
        rows in all (with cu; default cu[-1], which waits for the GPU). Positions outside the cache
        read as NaN; rows behind the last sequence's are not set."""
        c, b = self._layer(layer, table)
        if dtype not in (torch.bfloat16, torch.float32):
            raise TypeError("dtype must be bfloat16 or float32")
        p = self._ints(pos, "pos", b)
        u = None if cu is None else self._ints(cu, "cu", b + 1)
        n = b if cu is None else int(cu[-1]) if total is None else total
        shape = (max(n, 0), self.n_kv_heads, self.head_dim)
        k = torch.empty(shape, dtype=dtype, device=self.device)
        v = torch.empty_like(k)
        if n > 0:
            self._call("q4nx_kv4_read", c, k.data_ptr(), v.data_ptr(), int(dtype == torch.float32), n, p,
                      u, 1 if cu is None else max_new or n, ops._stream())
        return k, v

    # ------------------------------------------------------------ attention
    def attn(self, layer: int, q: torch.Tensor, lens: torch.Tensor | None = None,
             cu: torch.Tensor | None = None, max_new: int | None = None, max_len: int | None = None,
             scale: float | None = None, sel: torch.Tensor | None = None, n_split: int = 0,
             out: torch.Tensor | None = None, want_f32: bool = False, ws: ops.Workspace | None = None,
             table: torch.Tensor | None = None):
        """GQA attention of q (bf16 [rows, Hq, D]) over the cache, bf16 [rows, Hq, D] (and the fp32
        copy when want_f32). One token per sequence, at position lens[b] - 1; or, with cu (int32
        [n_seqs + 1]), a block of new tokens each, causal, the last at lens[b] - 1 (max_new: the most
        of one sequence; no result hangs on it). lens counts the new tokens, whose rows the cache
        holds already. max_len: at least the longest length (fewer read fewer positions). scale:
        default D ** -0.5. sel: `select`'s pages, for one token per sequence. out: rows behind the
        last sequence are left as they are."""
        c, b = self._layer(layer, table)
        n, hq, stride = self._query(q)
        d = self.head_dim
        lp = self._ints(self.lens if lens is None else lens, "lens", b)
        u = None if cu is None else self._ints(cu, "cu", b + 1)
        if cu is None and n != b:
            raise ValueError(f"{n} rows for {b} sequences (give cu for other numbers of rows)")
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
        else:
            self._tensor(out, "out", torch.bfloat16)
            if out.shape != q.shape or not out.is_contiguous():
                raise ValueError("out must be contiguous, of q's shape")
        of = torch.empty((n, hq, d), dtype=torch.float32, device=self.device) if want_f32 else None
        if n == 0:
            return (out, of) if want_f32 else out
        sp, ns = None, 0
        if sel is not None:
            self._tensor(sel, "sel", torch.int32)
            if sel.dim() != 3 or sel.shape[:2] != (b, self.n_kv_heads) or not sel.is_contiguous() \
                    or sel.shape[2] == 0:
                raise ValueError(f"sel must be [{b}, {self.n_kv_heads}, pages]")
            sp, ns = sel.data_ptr(), sel.shape[2]
        new = 1 if cu is None else max_new or n
        most = self._most(c, max_len)
        if most == 0:   # the library wants one position at least: the lengths are zeros instead
            none = torch.zeros(b, dtype=torch.int32, device=self.device)
            most, lp = 1, none.data_ptr()
        need = self._need(c, "q4nx_kv4_attn_ws_bytes", hq, 0 if cu is None else n, new, most, ns, n_split)
        wp = wn = 0
        if need:
            ws, wp, wn, stream = ops._scratch(ws, need)
        else:
            stream = ops._stream()
        self._call("q4nx_kv4_attn", c, q.data_ptr(), stride, out.data_ptr(),
                   None if of is None else of.data_ptr(), hq, u, n, new, lp, most,
                   d ** -0.5 if scale is None else float(scale), sp, ns, int(n_split), wp or None, wn,
                   stream)
        return (out, of) if want_f32 else out

    def select(self, layer: int, q: torch.Tensor, lens: torch.Tensor | None = None, n_sel: int = 64,
               n_first: int = 1, n_last: int = 1, max_len: int | None = None,
               out: torch.Tensor | None = None, ws: ops.Workspace | None = None,
               table: torch.Tensor | None = None) -> torch.Tensor:
        """The n_sel logical pages per (sequence, kv head) that q (one token per sequence) scores
        highest, int32 [n_seqs, Hkv, n_sel], ascending, -1 behind the last; the first n_first and the
        last n_last of a sequence are always among them."""
        c, b = self._layer(layer, table)
        n, hq, stride = self._query(q)
        if n != b:
            raise ValueError(f"{n} rows for {b} sequences")
        lp = self._ints(self.lens if lens is None else lens, "lens", b)
        if out is None:
            out = torch.empty((b, self.n_kv_heads, n_sel), dtype=torch.int32, device=self.device)
        else:
            self._tensor(out, "out", torch.int32)
            if out.shape != (b, self.n_kv_heads, n_sel) or not out.is_contiguous():
                raise ValueError(f"out must be contiguous [{b}, {self.n_kv_heads}, {n_sel}]")
        most = self._most(c, max_len)
        if most == 0:   # the library wants one position at least: the lengths are zeros instead
            none = torch.zeros(b, dtype=torch.int32, device=self.device)
            most, lp = 1, none.data_ptr()
        ws, wp, wn, stream = ops._scratch(ws, self._need(c, "q4nx_kv4_select_ws_bytes", most))
        self._call("q4nx_kv4_select", c, q.data_ptr(), stride, hq, lp, most, n_sel, n_first, n_last,
                   out.data_ptr(), wp, wn, stream)
        return out

    # ------------------------------------------------------------ pages
    def _pages_ws(self, n: int, ws):
        c, _ = self._layer(0, None)
        ws, wp, wn, stream = ops._scratch(ws, self._need(c, "q4nx_kv4_pages_ws_bytes", n))
        return c, ws, wp, wn, stream

    def reserve(self, want, ws: ops.Workspace | None = None) -> None:
        """Gives every sequence the pages it lacks for want[b] positions, the lowest free ones in the
        order of the sequences; `status`: sequences whose pages do not all fit (they get none)."""
        want = self._list(want, "want")
        if want.shape[0] != self.n_seqs:
            raise ValueError(f"want needs {self.n_seqs} values")
        c, ws, wp, wn, stream = self._pages_ws(0, ws)
        self._call("q4nx_kv4_reserve", c, self.refs.data_ptr(), want.data_ptr(), self.status.data_ptr(),
                  wp, wn, stream)

    def fork(self, src, dst, ws: ops.Workspace | None = None) -> None:
        """Sequence dst[i] (one without pages) goes on from src[i]: full pages shared, the last one
        copied in every layer. `status`: pairs that were not done."""
        src, dst = self._list(src, "src"), self._list(dst, "dst")
        n = src.shape[0]
        if dst.shape[0] != n or n > self.n_seqs:
            raise ValueError(f"src and dst must pair up, at most {self.n_seqs} of them")
        if n == 0:
            return
        c, ws, wp, wn, stream = self._pages_ws(n, ws)
        self._call("q4nx_kv4_fork", c, self.pool.stride(0), self.n_layers, self.lens.data_ptr(),
                  self.refs.data_ptr(), src.data_ptr(), dst.data_ptr(), n, self.status.data_ptr(), wp, wn,
                  stream)

    def free(self, seqs) -> None:
        """Gives the sequences' pages back and sets their lengths to 0."""
        seqs = self._list(seqs, "seqs")
        n = seqs.shape[0]
        if n > self.n_seqs:
            raise ValueError(f"at most {self.n_seqs} sequences")
        if n == 0:
            return
        c, _ = self._layer(0, None)
        self._call("q4nx_kv4_free", c, self.lens.data_ptr(), self.refs.data_ptr(), seqs.data_ptr(), n,
                  self.status.data_ptr(), ops._stream())

    def compact(self, ws: ops.Workspace | None = None) -> torch.Tensor:
        """Moves the pages in use to the front of the pool, tables with them; their number, int32 [1]
        on the device (pages from there on are free)."""
        live = torch.empty(1, dtype=torch.int32, device=self.device)
        c, ws, wp, wn, stream = self._pages_ws(0, ws)
        self._call("q4nx_kv4_compact", c, self.pool.stride(0), self.n_layers, self.refs.data_ptr(),
                  live.data_ptr(), wp, wn, stream)
        return live

    def copy_pages(self, src, dst) -> None:
        """Copies page src[i] to dst[i] in every layer (pages of the pool; tables and counts stay). No
        page may be written that another pair reads or writes."""
        src, dst = self._list(src, "src"), self._list(dst, "dst")
        if dst.shape[0] != src.shape[0]:
            raise ValueError("src and dst must pair up")
        if src.shape[0] == 0:
            return
        c, _ = self._layer(0, None)
        self._call("q4nx_kv4_copy_pages", c, self.pool.stride(0), self.n_layers, src.data_ptr(),
                  dst.data_ptr(), src.shape[0], ops._stream())
