"""Batched tree verification over a paged KV cache with a shared prefix.

``BatchKVCache`` reserves a whole capacity per sequence and holds a prompt that
all sequences start with (a system prompt, a document) once per sequence. Here
the K/V lie in pages of one pool, given to sequences as they grow, and the
shared prefix is held, and attended to, once for the batch:

- ``PagedKVCache``: pools [L][pages][nkv][page_size][hd], block tables, the
  free list (all on the device); ``set_prefix`` and ``load`` move prefilled
  ``TreeKVCache`` rows into pages, ``release`` returns a finished sequence's;
- ``forward_causal_paged``: the next tokens of every sequence's prompt, whose
  K/V stay (a chunked prefill);
- ``forward_tree_paged``: one pass over every sequence's tree, as
  ``forward_tree_batch`` over contiguous caches (per sequence
  ``forward_cached``, src/pe/target.py:203-224);
- ``commit_paged``: every sequence's accepted rows kept (src/pe/target.py:194-201
  with the keep index of src/pe/serve.py:308-309), as ``commit_batch``.

The walk between the two is ``batch.accept_batch_device``.
"""

from __future__ import annotations

import ctypes as C

import torch

from . import _lib, ops
from .batch import BatchTrees, tree_masks_batch
from .target import TargetModel, TreeKVCache


class PagedKVCache:
    """K/V pages of ``batch`` sequences. ``max_len`` bounds a sequence's tokens
    behind the shared prefix (the width of its block table)."""

    def __init__(self, target: TargetModel, batch: int, num_pages: int, page_size: int = 64, max_len: int = 4096):
        s, dev = target.shape, target.device
        if batch < 1 or num_pages < 1 or max_len < 1 or page_size not in (16, 32, 64, 128, 256, 512, 1024):
            raise ValueError("a paged cache needs sequences, pages and a page size of 16 to 1024 (a power of two)")
        self.shape, self.batch, self.num_pages, self.page_size = s, int(batch), int(num_pages), int(page_size)
        self.k = torch.zeros((s.num_layers, num_pages, s.num_kv_heads, page_size, s.head_dim), dtype=target.dtype,
                             device=dev)
        self.v = torch.zeros_like(self.k)
        i32 = {"dtype": torch.int32, "device": dev}
        self.block_table = torch.full((batch, -(-max_len // page_size)), -1, **i32)
        self.held = torch.zeros(batch, **i32)
        self.free_pages = torch.arange(num_pages - 1, -1, -1, **i32)
        self.free_top = torch.full((1,), num_pages, **i32)
        self.prefix_table = torch.empty(0, **i32)
        self.prefix_len = 0
        self.seq_lens = [0] * batch  # cached tokens of each sequence, the shared ones included
        self._status = target.status

    def pages_free(self) -> int:
        """Pages on the free list (waits for the device)."""
        return int(self.free_top.item())

    def slots(self, lens: torch.Tensor, row0: torch.Tensor, rows: int) -> torch.Tensor:
        """Pages for the rows [row0[b], row0[b + 1]) behind each sequence's lens[b] tokens, and their slots."""
        return ops.page_tables(lens, row0, self.block_table, self.held, self.free_pages, self.free_top, self.page_size,
                               rows, self._status, prefix_len=self.prefix_len)

    def set_prefix(self, cache: TreeKVCache) -> None:
        """Hold ``cache``'s rows as the prefix of every sequence (all of them empty)."""
        if self.prefix_len or any(self.seq_lens):
            raise ValueError("the prefix is set once, before any sequence holds tokens")
        n, dev = cache.seq_len, self.k.device
        if n == 0:
            return
        table = torch.full((1, -(-n // self.page_size)), -1, dtype=torch.int32, device=dev)
        held = torch.zeros(1, dtype=torch.int32, device=dev)
        slots = ops.page_tables(torch.zeros(1, dtype=torch.int64, device=dev),
                                torch.tensor([0, n], dtype=torch.int32, device=dev), table, held, self.free_pages,
                                self.free_top, self.page_size, n, self._status)
        self._write(cache, 0, n, slots)
        ops.read_status(self._status, "set_prefix")
        self.prefix_table, self.prefix_len = table.view(-1), n
        self.seq_lens = [n] * self.batch

    def load(self, b: int, cache: TreeKVCache) -> None:
        """Sequence ``b`` (empty behind the prefix) takes ``cache``'s rows from the prefix on."""
        n = cache.seq_len
        if self.seq_lens[b] != self.prefix_len or n < self.prefix_len:
            raise ValueError("load fills a sequence that is empty behind the prefix from a cache that covers it")
        rows, dev = n - self.prefix_len, self.k.device
        if rows == 0:
            return
        row0 = torch.tensor([0] * (b + 1) + [rows] * (self.batch - b), dtype=torch.int32, device=dev)
        lens = torch.tensor(self.seq_lens, dtype=torch.int64, device=dev)
        self._write(cache, self.prefix_len, n, self.slots(lens, row0, rows))
        ops.read_status(self._status, "load")
        self.seq_lens[b] = n

    def _write(self, cache: TreeKVCache, lo: int, hi: int, slots: torch.Tensor) -> None:
        ops.kv_write_paged(cache.k[:, :, lo:hi].transpose(1, 2), cache.v[:, :, lo:hi].transpose(1, 2), self.k, self.v,
                           slots, self._status)

    def release(self, *seqs: int) -> None:
        """Return the pages of finished sequences; they are empty behind the prefix afterwards."""
        if not all(0 <= b < self.batch for b in seqs) or len(set(seqs)) != len(seqs):
            raise ValueError("release names sequences of the cache, each once")
        ops.page_release(torch.tensor(seqs, dtype=torch.int32, device=self.k.device), self.block_table, self.held,
                         self.free_pages, self.free_top, self._status)
        for b in seqs:
            self.seq_lens[b] = self.prefix_len


def _forward(tm: TargetModel, cache: PagedKVCache, ids, pos, bits, words: int, seq_row0, seq_len, rows: int,
             max_rows: int, max_len: int, mask_mode: int, where: str) -> tuple[torch.Tensor, torch.Tensor]:
    dev, lib = tm.device, _lib.load()
    slots = cache.slots(seq_len, seq_row0, rows)
    logits = torch.empty((rows, tm.shape.vocab), dtype=tm.dtype, device=dev)
    fused = torch.empty((rows, tm.feature_dim), dtype=tm.dtype, device=dev)
    # the linears' arrival counters start at zero
    ws = torch.zeros(int(lib.pe_forward_paged_workspace_bytes(C.byref(tm.model.desc()), rows, max_rows, max_len,
                                                              cache.batch, cache.prefix_len)), dtype=torch.uint8,
                     device=dev)
    a = _lib.PassArgs()
    a.input_ids, a.positions, a.M, a.mask_mode, a.prefix_len = ids.data_ptr(), pos.data_ptr(), rows, mask_mode, max_len
    if bits is not None:
        a.tree_bits, a.bits_words = bits.data_ptr(), words
    fl = tm.feature_layers
    a.num_features = len(fl)
    for i, f in enumerate(fl[:4]):
        a.feature_layers[i] = f
    a.k_cache, a.v_cache = cache.k.data_ptr(), cache.v.data_ptr()
    a.logits, a.fused = logits.data_ptr(), fused.data_ptr()
    a.workspace, a.workspace_bytes, a.status = ws.data_ptr(), ws.numel(), tm.status.data_ptr()
    a.batch, a.max_seq_rows = cache.batch, max_rows
    a.seq_row0, a.seq_prefix = seq_row0.data_ptr(), seq_len.data_ptr()
    a.slots, a.block_table = slots.data_ptr(), cache.block_table.data_ptr()
    a.prefix_table = cache.prefix_table.data_ptr() if cache.prefix_len else None
    a.ld_table = a.table_cols = cache.block_table.shape[1]
    a.num_pages, a.prefix_pages, a.shared_len = cache.num_pages, cache.prefix_table.numel(), cache.prefix_len
    a.page_size = cache.page_size
    _lib.check(lib.pe_forward(C.byref(tm.model.desc()), C.byref(a), ops.stream_ptr()), where)
    ops.read_status(tm.status, where)
    return logits, fused


@torch.no_grad()
def forward_tree_paged(tm: TargetModel, node_tokens: list[list[int]], parents: list[list[int]],
                       cache: PagedKVCache) -> tuple[torch.Tensor, torch.Tensor, BatchTrees]:
    """Verify one tree per sequence in one pass (``forward_tree_batch`` over pages): (logits [M][V], fused [M][F],
    trees). The rows' K/V lie behind each sequence's cached tokens; the lengths change with ``commit_paged``."""
    if len(node_tokens) != cache.batch:
        raise ValueError("one tree per sequence of the cache")
    trees = BatchTrees(node_tokens, parents, cache.seq_lens, tm.device)
    bits, pos, _ = tree_masks_batch(trees, tm.status)
    logits, fused = _forward(tm, cache, trees.tokens, pos, bits, trees.words, trees.seq_row0, trees.seq_prefix, trees.M,
                             trees.max_rows, max(trees.prefix), _lib.PE_MASK_TREE, "forward_tree_paged")
    return logits, fused, trees


@torch.no_grad()
def forward_causal_paged(tm: TargetModel, tokens: list[list[int]],
                         cache: PagedKVCache) -> tuple[torch.Tensor, torch.Tensor, list[int]]:
    """Append each sequence's next tokens (an empty list: none) in one pass: (logits [M][V], fused [M][F], row0),
    sequence b's rows being row0[b] .. row0[b + 1] - 1. Their K/V stay cached."""
    if len(tokens) != cache.batch or not any(tokens):
        raise ValueError("one token list per sequence of the cache, not all empty")
    row0, flat, pos = [0], [], []
    for t, n in zip(tokens, cache.seq_lens):
        row0.append(row0[-1] + len(t))
        flat += [int(x) for x in t]
        pos += range(n, n + len(t))
    dev = tm.device
    logits, fused = _forward(tm, cache, torch.tensor(flat, dtype=torch.int64, device=dev),
                             torch.tensor(pos, dtype=torch.int64, device=dev), None, 0,
                             torch.tensor(row0, dtype=torch.int32, device=dev),
                             torch.tensor(cache.seq_lens, dtype=torch.int64, device=dev), row0[-1],
                             max(len(t) for t in tokens), max(cache.seq_lens), _lib.PE_MASK_CAUSAL,
                             "forward_causal_paged")
    cache.seq_lens = [n + len(t) for n, t in zip(cache.seq_lens, tokens)]
    return logits, fused, row0


def commit_paged(tm: TargetModel, cache: PagedKVCache, trees: BatchTrees, accept_out: torch.Tensor) -> None:
    """Keep each sequence's accepted path, moved together on the device (``commit_batch`` over pages); reads the path
    lengths back to set the cache's."""
    ops.kv_compact_paged(cache.k, cache.v, cache.block_table, trees.seq_prefix, accept_out, tm.status,
                         prefix_len=cache.prefix_len)
    lens = accept_out[:, 0].cpu().tolist()
    ops.read_status(tm.status, "commit_paged")
    cache.seq_lens = [p + int(n) for p, n in zip(trees.prefix, lens)]
