"""The engine over a 4-bit KV cache (Engine.build(kv_bits=4)): what its cache holds against the 16-bit
cache's rows, the prefill and decode kernels against each other through a whole model, snapshots, and
the refusals."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from hawking_b200.engine.checkpoint import load_sequence, save_sequence  # noqa: E402
from hawking_b200.engine.engine import Engine  # noqa: E402
from hawking_b200.engine.sampling import SamplingParams  # noqa: E402
from hawking_b200.formats.synth import random_prompt  # noqa: E402
from hawking_b200.models.config import preset  # noqa: E402
from hawking_b200.models.llama import random_llama_weights  # noqa: E402

SMALL = dict(layers=2, hidden=1024, ffn=2048, vocab=4096, max_ctx=512)
MODELS = {
    "q4k-128": preset("llama3-8b", n_heads=8, n_kv_heads=2, **SMALL),           # tensor-core GEMMs, bf16 attention rows
    "q4_0-64": preset("tiny-llama", layers=2, vocab=4096, max_ctx=512),         # dp4a GEMVs, int8 attention rows
    "qk-norm": preset("llama3-8b", n_heads=8, n_kv_heads=8, qk_norm=True, qkv_bias=True, rope_style=1, **SMALL),
}


@pytest.fixture(scope="module", params=list(MODELS))
def parts(request):
    cfg = MODELS[request.param]
    return cfg, random_llama_weights(cfg, "cuda", seed=3, std=0.05)


def _engine(parts, bits=4, **kw):
    cfg, w = parts
    kw = {**dict(max_batch=4, max_ctx=512, block_size=32, num_blocks=64, max_rows=64), **kw}
    return Engine.build(cfg, w, device="cuda", kv_bits=bits, **kw)


def test_cache_holds_the_16_bit_rows_to_half_a_step(parts):
    """Layer 0's keys and values do not depend on the cache: each is within half a quantisation step of
    the bf16 cache's (plus the float16 rounding of scale and centre, and the bf16 row's own rounding)."""
    toks = random_prompt(100, 4096, seed=2)
    e4, e16 = _engine(parts), _engine(parts, 16)
    for e in (e4, e16):
        e.model.forward_tokens(toks, seq_id=9)
    slots = torch.tensor(e16.kv.bm.slots(9, 0, 100), device="cuda")
    bs = e16.kv.block_size
    for got, full in zip(e4.kv.read(9, 0), (e16.kv.k[0], e16.kv.v[0])):
        want = full[slots // bs, :, slots % bs].double()
        g = want.reshape(100, want.shape[1], -1, 64)
        lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
        step = (hi - lo) / 15 * (1 + 2.0 ** -6)
        tol = 0.5 * step + 2.0 ** -10 * (lo.abs() + hi.abs() + 16 * step) + 2.0 ** -7 * g.abs()
        assert ((got.double().reshape(g.shape) - g).abs() <= tol).all()


def test_attention_rows_follow_from_the_cache(parts):
    """The model's attention rows of its last layer, recomputed in 64 bits from the cache it left and the
    queries it wrote."""
    import math
    cfg = parts[0]
    e = _engine(parts)
    m, kv = e.model, e.kv
    m.forward_tokens(random_prompt(150, 4096, seed=4), seq_id=1)  # one forward
    k, v = (t.double().repeat_interleave(cfg.n_heads // cfg.n_kv_heads, 1) for t in kv.read(1, cfg.layers - 1))
    q = m.q[:150].double()
    s = torch.einsum("rhd,thd->rht", q, k) / math.sqrt(cfg.head_dim)
    seen = torch.arange(150, device="cuda") <= torch.arange(150, device="cuda")[:, None]
    w = torch.softmax(s.masked_fill(~seen[:, None], -math.inf), -1)
    want = torch.einsum("rht,thd->rhd", w, v).reshape(150, -1)
    got = (m.attb if m.use_tensor_cores(150) else m.attf)[:150].double()
    # read() rounds keys and values to bf16: 2^-9 of each, of the scores by up to 2^-9 sum |q k|
    shift = (torch.einsum("rhd,thd->rht", q.abs(), k.abs()) / math.sqrt(cfg.head_dim) * 2.0 ** -9).amax()
    assert ((got - want).abs() <= v.abs().amax() * (2.0 ** -7 + 2 * shift)).all()
    assert (got - want).norm() <= 0.02 * want.norm()


def test_prefill_and_decode_kernels_agree_through_the_model(parts):
    """One step with a decoding sequence next to a prompt chunk: rows split over the two kernels, and all rows
    on the decode kernel. The kernels differ by float16 roundings of the attention's operands."""
    e = _engine(parts)
    m, kv = e.model, e.kv
    a, b = random_prompt(301, 4096, seed=5), random_prompt(140, 4096, seed=6)
    m.forward_tokens(a[:300], seq_id=1)
    m.forward_tokens(b[:100], seq_id=2)
    for s, n in ((1, 301), (2, 140)):
        assert kv.bm.reserve(s, n)
    kv.sync_tables([1, 2])
    ids = [a[300]] + b[100:140]
    out = []
    for long_runs in (True, False):
        m.inp.upload_plan(ids, [(kv.row(1), 300, 1), (kv.row(2), 100, 40)], kv, kv.ws.status)
        m.long_runs, m.decode_rows = long_runs, 1
        m.forward(41, "none")
        out.append(m.logits[:41].double().clone())
    m.long_runs = False
    assert m.inp.positions[:41].tolist() == [300] + list(range(100, 140))
    assert m.inp.row_ctx[:41].tolist() == [301] + list(range(101, 141))
    assert m.inp.slots[:41].tolist() == kv.bm.slots(1, 300, 301) + kv.bm.slots(2, 100, 140)
    assert kv.ws.status.item() == 0
    assert (out[0] - out[1]).abs().max() <= 3e-2 * out[1].abs().max()


def test_generates_batched_with_chunked_prefill(parts):
    prompts = [random_prompt(n, 4096, seed=n) for n in (5, 150, 64, 33, 1, 290)]
    e = _engine(parts, max_prefill_tokens=64)
    outs = e.generate(prompts, SamplingParams(max_tokens=12))
    assert [len(o) for o in outs] == [12] * 6
    # the continuation's first token follows from the prompt's teacher-forced logits where it is decided
    for p, o in zip(prompts, outs):
        lg = _engine(parts).model.forward_tokens(p, seq_id=3)[-1].double()
        assert lg.max() - lg[o[0]] <= 6e-2 * lg.abs().max()


def test_snapshot_restores_bit_for_bit(parts, tmp_path):
    toks = random_prompt(77, 4096, seed=8)
    e = _engine(parts)
    e.model.forward_tokens(toks[:76], seq_id=1)
    path = str(tmp_path / "s.kv")
    assert save_sequence(e.kv, 1, toks[:76], path)["dtype"] == "kv4"
    f = _engine(parts)
    f.model.forward_tokens(toks[:40], seq_id=5)  # other blocks are in use
    assert load_sequence(f.kv, 2, path) == toks[:76]
    for layer in range(e.cfg.layers):
        for x, y in zip(e.kv.read(1, layer, 76), f.kv.read(2, layer, 76)):
            assert torch.equal(x, y)
    with pytest.raises(ValueError, match="precision"):
        load_sequence(_engine(parts, 16).kv, 2, path)
    with pytest.raises(ValueError, match="block size"):
        load_sequence(_engine(parts, block_size=16).kv, 2, path)


def test_fork_copies_blocks(parts):
    e = _engine(parts)
    e.model.forward_tokens(random_prompt(32, 4096, seed=9), seq_id=1)
    src = e.kv.bm.table(1)[0]
    dst = next(b for b in range(64) if b not in e.kv.bm.table(1))
    e.kv.copy_blocks([(src, dst)])
    assert torch.equal(e.kv.data[:, src], e.kv.data[:, dst]) and e.kv.data[:, dst].any()


def test_refusals(parts):
    with pytest.raises(ValueError, match="16 or 4"):
        _engine(parts, 8)
    with pytest.raises(ValueError, match="multiple of 16"):
        _engine(parts, block_size=8)
    with pytest.raises(ValueError, match="16-bit KV cache"):
        _engine(parts).enable_speculative(4)
    e = _engine(parts)
    assert e.kv.data.numel() * 32 == _engine(parts, 16).kv.k.numel() * 2 * 2 * 9
    # a sequence row outside the tables: the step fails before any token is committed
    e.model.inp.upload_plan([1, 2], [(99, 0, 2)], e.kv, e.kv.ws.status)
    with pytest.raises(RuntimeError, match="bad argument"):
        e._check_device_status()
    e.clear_device_status()
    e._check_device_status()
