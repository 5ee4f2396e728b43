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


def _bytes_of(token, hd):
    """The bytes of a unit that hold token ``token``, by the format: key codes, value codes, pairs."""
    row, out = min(hd, 128) // 2, set()
    for d in range(hd):
        r, nib = d % 128, (d % 8) // 2 + 4 * (d % 2)
        out.add((d // 128) * 16 * row + token * row + ((r // 8) % 4) * (row // 4) + (r // 32) * 4 + nib // 2)
        r, nib = d % 64, (d % 4) + 4 * (token % 2)
        out.add(8 * hd + (d // 64) * 512 + ((r % 32) // 4) * 64 + ((token % 8) // 2) * 16 + (r // 32) * 8
                + (token // 8) * 4 + nib // 2)
        for value in (0, 1):
            out |= {(16 + value) * hd + token * (hd // 16) + (d // 64) * 4 + i for i in range(4)}
    return sorted(out)


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_every_byte_of_a_unit_is_one_tokens(hd):
    of = torch.full((18 * hd,), -1)
    for t in range(16):
        assert (of[_bytes_of(t, hd)] == -1).all()
        of[_bytes_of(t, hd)] = t
    assert (of >= 0).all()
    assert torch.equal(kv4.unit_tokens(hd), of)


@pytest.mark.parametrize("hd,bs,n", [(64, 16, 17), (64, 48, 35), (128, 16, 31), (128, 64, 64), (256, 32, 41), (64, 32, 1)])
def test_snapshots_hold_the_sequences_tokens_alone(tmp_path, hd, bs, n):
    """What another sequence left in the last block reaches neither the file nor its digest."""
    of = torch.full((18 * hd,), -1)
    for t in range(16):
        of[_bytes_of(t, hd)] = t
    of = 16 * torch.arange(bs // 16)[:, None] + of  # token of the block, of every byte
    live = torch.randint(0, 256, (2, -(-n // bs), 2, bs // 16, 18 * hd), dtype=torch.uint8)
    digests = []
    for i in range(2):
        kv = CpuKV4(2, 2, hd, 8, bs, 4, 8, "cpu", prefix_cache=False)
        kv.data.copy_(torch.randint(0, 256, kv.data.shape, dtype=torch.uint8))
        kv.bm.reserve(7, bs * i + 1)  # other blocks
        kv.bm.reserve(1, n)
        table = kv.bm.table(1)
        for b, blk in enumerate(table):
            mine = (of < n - b * bs).expand_as(live[:, b])
            kv.data[:, blk] = torch.where(mine, live[:, b], kv.data[:, blk])
        before = kv.data.clone()
        digests.append(save_sequence(kv, 1, list(range(n)), str(tmp_path / f"{i}.kv"))["payload_sha256"])
        assert torch.equal(kv.data, before)
    assert digests[0] == digests[1]
    kv = CpuKV4(2, 2, hd, 8, bs, 4, 8, "cpu", prefix_cache=False)
    kv.data.fill_(255)
    assert load_sequence(kv, 3, str(tmp_path / "0.kv")) == list(range(n))
    for b, blk in enumerate(kv.bm.table(3)):
        mine = (of < n - b * bs).expand_as(live[:, b])
        assert torch.equal(kv.data[:, blk], torch.where(mine, live[:, b], 0))
