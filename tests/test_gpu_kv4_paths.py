"""Ways through the framework that reach the 4-bit KV cache: an MoE model, shared prompt prefixes in memory and on
disk, and the command line."""
import json
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from hawking_b200.engine.engine import Engine  # noqa: E402
from hawking_b200.engine.sampling import SamplingParams  # noqa: E402
from hawking_b200.formats.synth import random_prompt  # noqa: E402
from hawking_b200.models.config import ModelConfig, preset  # noqa: E402
from hawking_b200.models.llama import random_llama_weights  # noqa: E402

DENSE = preset("tiny-llama", layers=2, vocab=4096, max_ctx=512)
MOE = ModelConfig(arch="mixtral", vocab=1024, hidden=512, layers=2, n_heads=8, n_kv_heads=2, head_dim=64, ffn=1024,
                  n_experts=4, top_k=2, expert_ffn=1024, weight_type="Q8_0", max_ctx=512)


@pytest.fixture(scope="module", params=["dense", "moe"])
def parts(request):
    cfg = DENSE if request.param == "dense" else MOE
    return cfg, random_llama_weights(cfg, "cuda", seed=5, std=0.05)


def _engine(parts, bits=4, **kw):
    return Engine.build(parts[0], parts[1], device="cuda", kv_bits=bits,
                        **{**dict(max_batch=4, max_ctx=512, block_size=32, num_blocks=64, max_rows=64), **kw})


def test_attention_rows_follow_from_the_cache(parts):
    """The last layer's attention rows, recomputed in 64 bits from the cache and the queries the model left."""
    cfg, n = parts[0], 120
    e = _engine(parts)
    m, kv = e.model, e.kv
    m.forward_tokens(random_prompt(n, cfg.vocab, seed=4), seq_id=1)
    k, v = (t.double().repeat_interleave(cfg.n_heads // cfg.n_kv_heads, 1) for t in kv.read(1, cfg.layers - 1))
    q = m.q[:n].double()
    s = torch.einsum("rhd,thd->rht", q, k) / math.sqrt(cfg.head_dim)
    seen = torch.arange(n, device="cuda") <= torch.arange(n, device="cuda")[:, None]
    want = torch.einsum("rht,thd->rhd", torch.softmax(s.masked_fill(~seen[:, None], -math.inf), -1), v).reshape(n, -1)
    got = (m.attb if m.use_tensor_cores(n) else m.attf)[:n].double()
    # read() rounds keys and values to bf16: 2^-9 of each, of the scores by up to 2^-9 sum |q k|
    shift = (torch.einsum("rhd,thd->rht", q.abs(), k.abs()) / math.sqrt(cfg.head_dim) * 2.0 ** -9).amax()
    assert ((got - want).abs() <= v.abs().amax() * (2.0 ** -7 + 2 * shift)).all()
    assert kv.ws.status.item() == 0


def test_a_batch_generates(parts):
    e = _engine(parts, max_prefill_tokens=64)
    outs = e.generate([random_prompt(n, parts[0].vocab, seed=n) for n in (5, 130, 33, 1, 64)], SamplingParams(max_tokens=9))
    assert [len(o) for o in outs] == [9] * 5
    assert all(0 <= t < parts[0].vocab for o in outs for t in o)


def test_a_shared_prefix_is_the_same_bytes(parts):
    """A second prompt takes the first one's blocks: its own prefill starts behind them and leaves them as they are."""
    vocab = parts[0].vocab
    head = random_prompt(96, vocab, seed=1)  # three blocks
    e = _engine(parts)
    first = e.add_request(head + random_prompt(20, vocab, seed=2), SamplingParams(max_tokens=4))
    e.step()
    blocks = e.kv.bm.table(first)[:3]
    before = e.kv.data[:, blocks].clone()
    second = e.add_request(head + random_prompt(31, vocab, seed=3), SamplingParams(max_tokens=4))
    rows = e.stats.prefill_rows
    e.step()
    assert e.kv.bm.table(second)[:3] == blocks
    assert e.stats.prefill_rows - rows <= 1 + 31  # (the first request's row, and what the second does not share)
    while e.has_work():
        e.step()
    assert torch.equal(e.kv.data[:, blocks], before)
    assert [len(e.requests[r].output) for r in (first, second)] == [4, 4]


def test_engines_of_both_precisions_share_a_prefix_directory(parts, tmp_path):
    vocab = parts[0].vocab
    prompt = random_prompt(97, vocab, seed=7)
    for bits, bs in ((16, 32), (4, 32), (4, 16)):
        for turn in range(2):
            e = _engine(parts, bits, block_size=bs)
            e.enable_prefix_disk(str(tmp_path), min_blocks=1)
            out = e.generate([prompt], SamplingParams(max_tokens=3))
            assert len(out[0]) == 3
            assert e.stats_disk == {"hits": turn, "hit_tokens": 96 * turn, "stored": 1 - turn}, (bits, bs, turn)


def test_generate_on_the_command_line(capsys):
    from hawking_b200.__main__ import main
    args = ["generate", "--preset", "tiny-llama", "--layers", "2", "--prompt", "hello", "--max-tokens", "4", "--max-ctx",
            "128", "--json", "--kv-bits"]
    for bits in ("4", "16"):
        assert main(args + [bits]) == 0
        assert 1 <= len(json.loads(capsys.readouterr().out)["tokens"]) <= 4
