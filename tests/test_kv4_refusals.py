"""Where the 4-bit KV cache is asked for and cannot be had: the call says so, and says it before any weights are
read (no GPU)."""
from types import SimpleNamespace

import pytest

from hawking_b200.engine.engine import Engine
from hawking_b200.engine.speculative import SpeculativeDecoder


def _engine(bits):
    """What the speculative entry points look at before they do anything."""
    model = SimpleNamespace(max_rows=64)
    return SimpleNamespace(kv=SimpleNamespace(bits=bits), model=model, spec=None, max_prefill_tokens=64)


def test_speculative_decoding_is_refused_at_every_entry_point():
    """A row's rounding over the 4-bit cache depends on the batch: the output would not be the greedy one."""
    eng = _engine(4)
    for call in (lambda: SpeculativeDecoder(eng), lambda: Engine.generate_speculative(eng, [1, 2, 3]),
                 lambda: Engine.enable_speculative(eng, 4)):
        with pytest.raises(ValueError, match="16-bit KV cache"):
            call()
    Engine.enable_speculative(eng, 0)  # turning it off is always right
    assert SpeculativeDecoder(_engine(16), k=3).k == 3
    Engine.enable_speculative(_engine(16), 4)
    assert SpeculativeDecoder(SimpleNamespace(kv=SimpleNamespace())).k == 4  # caches that state no precision hold 16 bits
