"""Shapes and sizes of the 4-bit KV cache (no GPU)."""
import pytest

from hawking_b200.config import EngineConfig
from hawking_b200.engine.kv_cache import PagedKV4Cache, PagedKVCache
from hawking_b200.ops import kv4


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_nine_bits_for_two_values(hd):
    assert kv4.unit_bytes(hd) * 8 == 16 * 2 * hd * 4.5
    assert kv4.cache_shape(7, 2, 48, hd) == (7, 2, 3, 18 * hd)
    a, b = (c.bytes_per_block(4, 2, hd, 64) for c in (PagedKV4Cache, PagedKVCache))
    assert a * 32 == b * 9


@pytest.mark.parametrize("hd,bs", [(32, 16), (96, 16), (512, 16), (64, 0), (64, 8), (64, 24), (64, -16)])
def test_refused_shapes(hd, bs):
    with pytest.raises(ValueError):
        kv4.cache_shape(1, 1, bs, hd)


def test_engine_config_passes_the_precision():
    assert EngineConfig().build_kwargs()["kv_bits"] == 16
    assert EngineConfig(kv_bits=4).build_kwargs()["kv_bits"] == 4
