"""Where the 4-bit KV cache is asked for and cannot be had: the call says so, and says it before any weights are
read (no GPU)."""
import json
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


# ---- models whose cache has 16 bits only ---------------------------------------------------------
@pytest.fixture
def no_weights(monkeypatch):
    """Every way to weights, made to fail: a refusal comes before them."""
    import torch

    from hawking_b200.models import deepseek, deepseek_gguf, qwen_next, qwen_next_artifact

    def reached(*a, **k):
        raise AssertionError("weights were read")

    for mod, name in ((deepseek, "random_deepseek_weights"), (deepseek_gguf, "load_deepseek_weights"),
                      (qwen_next, "random_qwen_next_weights"), (qwen_next_artifact, "load"),
                      (torch.cuda, "mem_get_info")):
        monkeypatch.setattr(mod, name, reached)


def _paths(tmp_path):
    """A deepseek2 GGUF file, and the index of a .gravity artifact of the hybrid architecture."""
    from hawking_b200.formats.synth import write_deepseek2_gguf
    from hawking_b200.models.config import preset
    cfg = preset("deepseek-v3").with_(vocab=1024, hidden=512, layers=2, n_heads=4, n_kv_heads=4, ffn=512, n_experts=4,
                                      top_k=2, expert_ffn=256, shared_ffn=256, n_groups=2, topk_groups=1,
                                      first_dense_layers=1, q_lora_rank=256, max_ctx=512, weight_type="Q4_K")
    gguf = write_deepseek2_gguf(str(tmp_path / "ds.gguf"), cfg)
    art = tmp_path / "a.gravity"
    art.mkdir()
    (art / "model.gravity.index.json").write_text(json.dumps({"architecture": {"name": "qwen3next"}}))
    return gguf, str(art)


def test_models_without_a_4_bit_cache_refuse_it(no_weights, tmp_path):
    from hawking_b200.serve.__main__ import path_engine, preset_engine
    gguf, art = _paths(tmp_path)
    calls = [lambda b: Engine.from_gguf(gguf, kv_bits=b), lambda b: Engine.from_path(gguf, kv_bits=b),
             lambda b: Engine.from_path(art, kv_bits=b), lambda b: path_engine(art, 1, kv_bits=b),
             lambda b: preset_engine("deepseek-v3", 1, kv_bits=b), lambda b: preset_engine("qwen3-next", 1, kv_bits=b)]
    for call in calls:
        with pytest.raises(ValueError, match="16-bit cache only"):
            call(4)
        with pytest.raises(ValueError, match="16 or 4"):
            call(8)
        with pytest.raises(AssertionError, match="weights were read"):  # 16 is what they have
            call(16)


def test_generate_refuses_before_it_loads(no_weights, tmp_path, capsys):
    from hawking_b200.__main__ import main
    gguf, art = _paths(tmp_path)
    for model in (["--gguf", gguf], ["--model", art], ["--preset", "deepseek-v3"], ["--preset", "qwen3-next"]):
        assert main(["generate", *model, "--prompt", "x", "--kv-bits", "4"]) == 2
        assert "not available for this model's cache" in capsys.readouterr().err


# ---- heads and block sizes that the kernels do not take ------------------------------------------
@pytest.mark.parametrize("heads,block_size,why", [(dict(n_heads=34, n_kv_heads=2), 64, "at most 16 query heads"),
                                                  (dict(n_heads=20, n_kv_heads=8), 64, "at most 16 query heads"),
                                                  (dict(head_dim=96), 64, "head_dim"), (dict(), 8, "multiple of 16"),
                                                  (dict(), 24, "multiple of 16")])
def test_engine_build_refuses_what_the_kernels_do_not_take(monkeypatch, heads, block_size, why):
    """Before the pool is sized (8 tokens a block made its blocks 0 bytes) and before the first forward."""
    import torch

    from hawking_b200.models import llama
    from hawking_b200.models.config import preset
    from hawking_b200.serve.__main__ import preset_engine

    def reached(*a, **k):
        raise AssertionError("went on")

    monkeypatch.setattr(torch.cuda, "mem_get_info", reached)
    monkeypatch.setattr(llama, "random_llama_weights", reached)
    cfg = preset("llama3-8b").with_(**heads)
    with pytest.raises(ValueError, match=why):
        Engine.build(cfg, None, device="cpu", block_size=block_size, kv_bits=4)
    with pytest.raises(AssertionError):  # the 16-bit cache takes what it took
        Engine.build(cfg, None, device="cpu", block_size=block_size)
    if not heads:
        with pytest.raises(ValueError, match=why):
            preset_engine("llama3-8b", 1, kv_bits=4, block_size=block_size)
        with pytest.raises(AssertionError):
            preset_engine("llama3-8b", 1, block_size=block_size)


def test_bytes_per_block_refuses_a_block_of_no_units():
    from hawking_b200.engine.kv_cache import PagedKV4Cache
    for bs in (0, 8, 24):
        with pytest.raises(ValueError, match="multiple of 16"):
            PagedKV4Cache.bytes_per_block(2, 2, 64, bs)
