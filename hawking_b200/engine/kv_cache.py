"""Paged KV cache storage on the device.

``PagedKVCache``: one bf16 tensor per K and V, [layers, num_blocks, n_kv_heads, block_size, head_dim].
A block holds ``block_size`` consecutive tokens of one sequence; each head's tokens inside a block are
contiguous so the decode kernel reads whole rows. ``PagedKV4Cache``: the same pool in 4 bits (ops/kv4.py),
one uint8 tensor at 9/32 of the bytes. Block allocation, prefix sharing and copy-on-write live in
the C++ ``BlockManager``; this class owns the memory and the device-side block tables.
"""
from __future__ import annotations

import math
from typing import Dict, Iterable, List, Optional, Tuple

import torch

from .._ext import native


class KVBitsError(ValueError):
    """A cache precision that a model cannot have."""


def check_kv_bits(bits: int, arch: str, cfg=None, block_size: int = 64) -> None:
    """Refuse a cache precision that does not exist, that the models of ``arch`` have no cache in, or whose
    kernels do not take the heads of ``cfg`` or the block size."""
    if bits not in (4, 16):
        raise KVBitsError(f"kv_bits must be 16 or 4, not {bits}")
    if bits != 16 and arch in ("deepseek2", "qwen3next"):
        raise KVBitsError(f"kv_bits={bits}: the models of architecture {arch} have a 16-bit cache only")
    if bits == 4 and cfg is not None:
        from ..ops import kv4
        if cfg.n_heads % cfg.n_kv_heads or cfg.n_heads // cfg.n_kv_heads > kv4.MAX_GROUP:
            raise KVBitsError(f"4-bit KV cache: a kv head serves at most {kv4.MAX_GROUP} query heads "
                              f"({cfg.n_heads} query heads, {cfg.n_kv_heads} kv heads)")
        try:
            kv4.cache_shape(1, cfg.n_kv_heads, block_size, cfg.head_dim)
        except ValueError as e:
            raise KVBitsError(str(e)) from None


class PagedKVCache:
    bits = 16

    def __init__(self, layers: int, n_kv_heads: int, head_dim: int, num_blocks: int, block_size: int,
                 max_seqs: int, max_blocks_per_seq: int, device, prefix_cache: bool = True,
                 dtype=torch.bfloat16):
        if num_blocks * block_size >= 2 ** 31:
            raise ValueError("KV pool too large for int32 slot ids")
        self.layers, self.nkv, self.hd = layers, n_kv_heads, head_dim
        self.num_blocks, self.block_size = num_blocks, block_size
        self._allocate(device, dtype)
        self.max_seqs, self.max_blocks = max_seqs, max_blocks_per_seq
        self.block_tables = torch.zeros(max_seqs, max_blocks_per_seq, dtype=torch.int32, device=device)
        self._host_tables = torch.zeros(max_seqs, max_blocks_per_seq, dtype=torch.int32).pin_memory() \
            if torch.cuda.is_available() else torch.zeros(max_seqs, max_blocks_per_seq, dtype=torch.int32)
        self.bm = native().BlockManager(num_blocks, block_size, prefix_cache)
        self._row_of: Dict[int, int] = {}
        self._free_rows: List[int] = list(range(max_seqs - 1, -1, -1))
        self._synced_len: Dict[int, int] = {}

    def _allocate(self, device, dtype):
        self.k = torch.zeros(self.layers, self.num_blocks, self.nkv, self.block_size, self.hd, dtype=dtype, device=device)
        self.v = torch.zeros_like(self.k)

    @property
    def device(self) -> torch.device:
        return self.block_tables.device

    @staticmethod
    def bytes_per_block(layers: int, n_kv_heads: int, head_dim: int, block_size: int, elem_bytes: int = 2) -> int:
        return 2 * layers * n_kv_heads * block_size * head_dim * elem_bytes

    # ---- table rows (one per live sequence) ----
    def row(self, seq_id: int) -> int:
        r = self._row_of.get(seq_id)
        if r is None:
            if not self._free_rows:
                raise RuntimeError("no free block-table rows")
            r = self._free_rows.pop()
            self._row_of[seq_id] = r
            self._synced_len[seq_id] = 0
        return r

    def drop(self, seq_id: int):
        r = self._row_of.pop(seq_id, None)
        if r is not None:
            self._free_rows.append(r)
        self._synced_len.pop(seq_id, None)
        if self.bm.has(seq_id):
            self.bm.release(seq_id)

    def sync_tables(self, seq_ids: Iterable[int]):
        """Copy changed block-table rows to the device."""
        for s in seq_ids:
            t = self.bm.table(s)
            if len(t) > self.max_blocks:
                raise RuntimeError("sequence exceeds max_blocks_per_seq")
            if self._synced_len.get(s, -1) == len(t):
                continue
            r = self.row(s)
            self._host_tables[r, : len(t)] = torch.tensor(t, dtype=torch.int32)
            self.block_tables[r].copy_(self._host_tables[r], non_blocking=True)
            self._synced_len[s] = len(t)

    def copy_blocks(self, pairs: List[Tuple[int, int]]):
        for src, dst in pairs:
            self.k[:, dst].copy_(self.k[:, src])
            self.v[:, dst].copy_(self.v[:, src])


class PagedKV4Cache(PagedKVCache):
    """The pool in 4 bits: ``data`` is uint8 [layers, num_blocks, n_kv_heads, block_size / 16,
    18 * head_dim] (ops/kv4.py describes a unit), ``ws`` what the attention launches share. The block
    size is a multiple of 16, the head dim 64, 128 or 256."""

    bits = 4

    def _allocate(self, device, dtype):
        from ..ops import kv4
        shape = kv4.cache_shape(self.num_blocks, self.nkv, self.block_size, self.hd)
        self.data = torch.zeros(self.layers, *shape, dtype=torch.uint8, device=device)
        self.ws = kv4.Workspace(device)

    @staticmethod
    def bytes_per_block(layers: int, n_kv_heads: int, head_dim: int, block_size: int, elem_bytes: int = 2) -> int:
        from ..ops import kv4
        return layers * math.prod(kv4.cache_shape(1, n_kv_heads, block_size, head_dim))

    def copy_blocks(self, pairs: List[Tuple[int, int]]):
        for src, dst in pairs:
            self.data[:, dst].copy_(self.data[:, src])

    def read(self, seq_id: int, layer: int, n: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """The first ``n`` (default: all) cached tokens' keys and values of one layer, as bf16
        [n, n_kv_heads, head_dim] rows: what attention reads, for a snapshot or a move to a 16-bit cache."""
        from ..ops import kv4
        n = self.bm.num_tokens(seq_id) if n is None else n
        slots = torch.tensor(self.bm.slots(seq_id, 0, n), dtype=torch.int32, device=self.device)
        k = torch.empty(n, self.nkv, self.hd, dtype=torch.bfloat16, device=self.device)
        v = torch.empty_like(k)
        kv4.gather(self.data[layer], slots, k, v)
        return k, v
