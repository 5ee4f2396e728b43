"""Snapshots of the 4-bit KV cache (engine/checkpoint.py) on CPU tensors; the same code runs on the GPU cache."""
import os

import pytest
import torch

from hawking_b200.engine.checkpoint import PrefixDiskCache, load_sequence, save_sequence
from hawking_b200.engine.kv_cache import PagedKV4Cache, PagedKVCache
from hawking_b200.ops import kv4


class CpuKV4(PagedKV4Cache):
    """The pool without the GPU's workspace."""

    def _allocate(self, device, dtype):
        self.data = torch.zeros(self.layers, *kv4.cache_shape(self.num_blocks, self.nkv, self.block_size, self.hd),
                                dtype=torch.uint8, device=device)


def _cache(bits, bs=16):
    return (CpuKV4 if bits == 4 else PagedKVCache)(2, 2, 64, 16, bs, 4, 8, "cpu", prefix_cache=False)


def test_one_directory_serves_both_precisions_and_any_block_size(tmp_path):
    """A snapshot of another kind is neither a hit nor in the way of one's own."""
    toks = list(range(5, 37))
    kinds = [(16, 16), (4, 16), (4, 32)]
    paths = []
    for bits, bs in kinds:
        kv = _cache(bits, bs)
        pc = PrefixDiskCache(str(tmp_path), kv=kv)
        assert pc.longest_prefix(toks) is None
        kv.bm.reserve(1, len(toks))
        p = pc.store(kv, 1, toks)
        assert os.path.exists(p) and p not in paths
        paths.append(p)
    for (bits, bs), p in zip(kinds, paths):
        kv = _cache(bits, bs)
        n, found = PrefixDiskCache(str(tmp_path), kv=kv).longest_prefix(toks + [1])
        assert (n, found) == (len(toks), p)
        assert load_sequence(kv, 2, found) == toks
    # 16-bit snapshots keep the name they had
    assert os.path.basename(paths[0]) == PrefixDiskCache.key(toks) + ".hkkv"
    assert PrefixDiskCache(str(tmp_path)).longest_prefix(toks) == (len(toks), paths[0])
