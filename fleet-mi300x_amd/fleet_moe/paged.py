"""Several sequences' latent cache in pages of 8-bit rows (fleet_cache_*), beside
`ops.Decoder`'s contiguous bf16 cache of one sequence.

A page holds 64 positions of every layer, in e4m3 with a power-of-two scale for
each block of 16 positions and part of a row (c, k_pe): 578 bytes a position and
layer instead of 1152. Sequences share pages: `remap` reorders, forks and frees
them by table entries alone, `grow` gives them room for new positions and copies a
page that two of them would write, `append` and `read` convert rows from and to
`Decoder.cache`'s bf16 bits, `attend` runs the absorbed-MLA attention of any
number of query tokens per sequence, and `compact` moves the used pages to the
front of the pool. All state is on the device; no call reads it back, allocates
more than its outputs or synchronises, so a step can be captured in a HIP graph.
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _lib
from .ops import _int32, _need, _on, _own, _ptr, _same_device, _stream

ROW = _lib.CACHE_ROW
LORA = 512
PAGE = _lib.CACHE_PAGE_TOKENS
PAGE_BYTES = _lib.CACHE_PAGE_BYTES
# (qk_nope + qk_rope)^-0.5 * mscale(40, 0.707)^2 (src/host/reference_decode.py:
# 78-83, 197-203), the decode kernels' factor
SOFTMAX_SCALE = 192.0 ** -0.5 * (0.1 * 0.707 * math.log(40.0) + 1.0) ** 2


class PagedCache:
    """The pages, tables and workspace of `n_seqs` sequences.

    pool uint8 [n_pages][n_layers][36992], table int32 [n_seqs][max_pages]
    (-1 behind a sequence's last page), lens int32 [n_seqs], refs int32 [n_pages]
    (table entries that name a page). Calls on one cache must be ordered on
    one stream (they share the workspace)."""

    def __init__(self, pool: torch.Tensor, table: torch.Tensor, lens: torch.Tensor,
                 refs: torch.Tensor):
        if pool.dim() != 3 or pool.shape[2] != PAGE_BYTES or table.dim() != 2:
            raise ValueError(f"pool: expected uint8 [pages][layers][{PAGE_BYTES}] and a table "
                             f"[seqs][max_pages], got {tuple(pool.shape)}, {tuple(table.shape)}")
        self.n_pages, self.n_layers = int(pool.shape[0]), int(pool.shape[1])
        self.n_seqs, self.max_pages = int(table.shape[0]), int(table.shape[1])
        _need(pool, torch.uint8, pool.shape, "pool")
        _need(table, torch.int32, table.shape, "table")
        _need(lens, torch.int32, (self.n_seqs,), "lens")
        _need(refs, torch.int32, (self.n_pages,), "refs")
        _same_device(pool, table=table, lens=lens, refs=refs)
        self.pool, self.table, self.lens, self.refs = pool, table, lens, refs
        self.device = pool.device
        self._c = _lib.FleetCache(_ptr(pool), _ptr(table), _ptr(lens), _ptr(refs), self.n_pages,
                                  self.n_layers, self.n_seqs, self.max_pages)
        self._ref = ctypes.byref(self._c)
        n = _lib.load().fleet_cache_workspace_bytes(self.n_pages, self.n_seqs)
        if n == 0:
            raise ValueError(f"unsupported cache sizes: {self.n_pages} pages, "
                             f"{self.n_seqs} sequences")
        # only the header (status word, the last grow's refusal) has to start as zero
        self.workspace = torch.empty(n, dtype=torch.uint8, device=self.device)
        self.workspace[:256].zero_()
        self._ws = (self.workspace.data_ptr(), n)
        self._fn = {name: getattr(_lib.load(), name) for name, *_ in _lib.SYMBOLS
                    if name.startswith("fleet_cache_")}

    @classmethod
    def empty(cls, n_pages: int, n_seqs: int, max_pages: int, n_layers: int,
              device="cuda") -> "PagedCache":
        """A cache whose sequences hold nothing yet."""
        new = lambda v, *s: torch.full(s, v, dtype=torch.int32, device=device)  # noqa: E731
        pool = torch.empty((n_pages, n_layers, PAGE_BYTES), dtype=torch.uint8, device=device)
        return cls(pool, new(-1, n_seqs, max_pages), new(0, n_seqs), new(0, n_pages))

    def _call(self, name: str, *args, stream=None) -> None:
        with _on(self.device):
            rc = self._fn[name](self._ref, *args, *self._ws, _stream(stream))
        if rc:
            _lib.check(rc, name)

    def remap(self, parents: torch.Tensor, stream=None) -> None:
        """Sequence i becomes what sequence parents[i] (int32 [n_seqs]) was, or empty
        for -1; pages no sequence holds any more are free."""
        _need(parents, torch.int32, (self.n_seqs,), "parents")
        _same_device(self.pool, parents=parents)
        self._call("fleet_cache_remap", _ptr(parents), stream=stream)

    def grow(self, n_new: torch.Tensor, stream=None) -> None:
        """Room for n_new[s] (int32 [n_seqs]) more positions of every sequence, all or
        none (see status()): lens grows by it, append() then writes them. After a
        refusal append() writes nothing until a grow() succeeds; to go on, free
        sequences with remap(), clear_status() and grow again."""
        _need(n_new, torch.int32, (self.n_seqs,), "n_new")
        _same_device(self.pool, n_new=n_new)
        self._call("fleet_cache_grow", _ptr(n_new), stream=stream)

    def compact(self, stream=None) -> torch.Tensor:
        """Moves the used pages to the front; returns their number, int32 [1]."""
        with _own(stream):
            used = torch.empty(1, dtype=torch.int32, device=self.device)
        self._call("fleet_cache_compact", _ptr(used), stream=stream)
        return used

    def _rows(self, name, rows, start, layer, stream):
        if rows.dim() == 2:
            rows = rows.unsqueeze(0)
        if (not rows.is_cuda or rows.dtype != torch.int16 or rows.dim() != 3
                or rows.shape[2] != ROW or (rows.numel() and rows.stride(2) != 1)):
            raise ValueError(f"rows: expected device int16 (bf16 bits) [layers][rows][{ROW}] "
                             f"with unit column stride, got {rows.dtype} {tuple(rows.shape)}")
        layers, n = int(rows.shape[0]), int(rows.shape[1])
        if n == 0 or layers == 0:
            return
        self._check_start(start, n)
        _same_device(self.pool, rows=rows, start=start)
        row = int(rows.stride(1)) if n > 1 else ROW
        step = int(rows.stride(0)) if layers > 1 else 0
        self._call(name, _int32(layer), layers, _ptr(rows), row, step, _ptr(start), n, stream=stream)

    def _check_start(self, start, n: int) -> None:
        if start is not None:
            _need(start, torch.int32, (self.n_seqs + 1,), "start")
        elif n != self.n_seqs:
            raise ValueError(f"without start there is one row per sequence: got {n}, "
                             f"{self.n_seqs} sequences")

    def append(self, rows: torch.Tensor, start: torch.Tensor | None = None, layer: int = 0,
               stream=None) -> None:
        """Writes each sequence's newest positions of layers layer, layer + 1, ..:
        rows int16 (bf16 bits) [layers][n][576] or [n][576], any layer and row
        strides that are multiples of 8; start int32 [n_seqs + 1]: sequence s
        gets rows start[s] .. start[s + 1] - 1 as its last positions. None: a row
        each."""
        self._rows("fleet_cache_append", rows, start, layer, stream)

    def read(self, rows: torch.Tensor, start: torch.Tensor | None = None, layer: int = 0,
             stream=None) -> None:
        """The reverse of append(): fills rows with the values the pages hold."""
        self._rows("fleet_cache_read", rows, start, layer, stream)

    def attend(self, q: torch.Tensor, start: torch.Tensor | None = None, layer: int = 0,
               max_len: int = 0, window: int = 0, sinks: int = 0,
               scale: float = SOFTMAX_SCALE, out: torch.Tensor | None = None,
               lse: torch.Tensor | None = None, stream=None):
        """Attention of q int16 (bf16 bits) [n][heads][576] over the cache's layer:
        tokens start[s] .. start[s + 1] - 1 stand at the last positions of sequence
        s (None: one token each). A token sees the positions up to its own; with
        window > 0 the last `window` of them and the first `sinks`. max_len: a
        bound on lens known to the caller, for the division of the work.
        Returns (out int16 [n][heads][512], lse fp32 [n][heads]), the given
        tensors or new ones."""
        if (not q.is_cuda or q.dtype != torch.int16 or q.dim() != 3 or q.shape[2] != ROW
                or (q.numel() and (q.stride(2) != 1 or (q.shape[1] > 1 and q.stride(1) != ROW)))):
            raise ValueError(f"q: expected device int16 (bf16 bits) [tokens][heads][{ROW}] with "
                             f"contiguous heads, got {q.dtype} {tuple(q.shape)}")
        n, heads = q.shape[0], q.shape[1]
        if out is not None:
            _need(out, torch.int16, (n, heads, LORA), "out")
        if lse is not None:
            _need(lse, torch.float32, (n, heads), "lse")
        if n:
            self._check_start(start, n)
        _same_device(self.pool, q=q, start=start, out=out, lse=lse)
        if out is None or lse is None:
            with _own(stream):
                if out is None:
                    out = torch.empty((n, heads, LORA), dtype=torch.int16, device=self.device)
                if lse is None:
                    lse = torch.empty((n, heads), dtype=torch.float32, device=self.device)
        if n == 0:
            return out, lse
        stride = q.stride(0) if n > 1 else heads * ROW
        self._call("fleet_cache_attend", _int32(layer), _ptr(q), stride, _ptr(start), n, heads,
                   _int32(max_len), _int32(window), _int32(sinks), float(scale), _ptr(out),
                   _ptr(lse), stream=stream)
        return out, lse

    def status(self, stream=None) -> int:
        """The FLEET_MOE_ABORT_* bits the calls left; synchronises."""
        v = ctypes.c_uint32(0)
        with _on(self.device):
            rc = _lib.load().fleet_moe_workspace_status(_ptr(self.workspace), ctypes.byref(v),
                                                        _stream(stream))
        _lib.check(rc, "fleet_moe_workspace_status")
        return int(v.value)

    def clear_status(self, stream=None) -> None:
        """Forgets the bits that status() collected, on the device."""
        with _on(self.device), _own(stream):
            self.workspace[8:12].zero_()
