"""The 4-bit KV cache's operators (ops/kv4.py) on what a caller can get wrong or a launch can fail at:
rows without a place, numbers at the end of int32, inputs that a kernel must not be given."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from hawking_b200.ops import kv4  # noqa: E402

DEV = "cuda"


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _plan(seq, cached, new, tab, bs, cap, free=None):
    """(rows, tables, blocks taken, status)."""
    out = torch.full((4, cap), 77, dtype=torch.int32, device=DEV)
    t, taken, status = _ints(tab) if isinstance(tab, list) else tab, _ints([-5]), _ints([0])
    kv4.plan_rows(_ints(seq), _ints(cached), _ints(new), t, bs, *out.unbind(0),
                  free_blocks=None if free is None else _ints(free), taken=taken, status=status)
    torch.cuda.synchronize()
    return out.t().tolist(), t, taken.item(), status.item()


# ---- rows without a place ------------------------------------------------------------------------
def test_plan_reports_rows_without_a_block():
    """A negative table entry leaves a row without a slot: the step's status says so."""
    for free in (None, [9, 8]):  # complete tables, and the partial block of a request that also takes new ones
        tab = [[5, -1, 7], [4, 6, 0]]
        rows, _, taken, status = _plan([0, 1], [30, 16], [2, 1], tab, 16, 3, free)
        assert rows == [[30, 0, 31, -1], [31, 0, 32, -1], [16, 1, 17, 96 if free is None else 144]]
        assert status == 4 and taken == (0 if free is None else 1)
    rows, _, _, status = _plan([0], [15], [2], [[5, -1, 7]], 16, 2)
    assert rows == [[15, 0, 16, 95], [16, 0, 17, -1]] and status == 4
    rows, _, _, status = _plan([0], [16], [1], [[5, 0, 0]], 16, 1, [-3])  # a block list's entry
    assert rows == [[16, 0, 17, -1]] and status == 4
    # an entry that no live row looks up does not matter
    assert _plan([0], [15], [1], [[5, -1, 7]], 16, 2)[3] == 0


def test_plan_reports_blocks_past_int32_slots():
    """block * block_size past 2^31 is no slot (in 32 bits it would come out as another valid one)."""
    for blk in (1 << 27, (1 << 28) + 3, 2 ** 31 - 1):
        rows, _, _, status = _plan([0, 1], [0, 3], [1, 1], [[blk, 0], [6, 0]], 16, 2)
        assert rows == [[0, 0, 1, -1], [3, 1, 4, 99]] and status == 4
    rows, _, _, status = _plan([0], [0], [16], [[(1 << 27) - 1, 0]], 16, 16)  # the last block of all
    assert status == 0 and [r[3] for r in rows] == list(range(2 ** 31 - 16, 2 ** 31))


def test_plan_lengths_near_2_to_the_31():
    """A table row whose last block ends just below 2^31 tokens: blocks are counted without passing int32."""
    bs, width = 65535, 32768
    tab = torch.full((3, width), 11, dtype=torch.int32, device=DEV)
    last = (width - 1) * bs
    rows, t, taken, status = _plan([2, 0, 1], [last, width * bs - 1, 0], [bs, 1, 1], tab.clone(), bs, bs + 2, [5, 4, 3])
    assert status == 0 and taken == 2
    assert rows[0] == [last, 2, last + 1, 5 * bs] and rows[bs - 1] == [last + bs - 1, 2, last + bs, 5 * bs + bs - 1]
    assert rows[bs:] == [[width * bs - 1, 0, width * bs, 11 * bs + bs - 1], [0, 1, 1, 4 * bs]]
    want = tab.clone()
    want[2, -1], want[1, 0] = 5, 4
    assert torch.equal(t, want)
    # one token past the row's end gets no rows
    assert _plan([0], [width * bs], [1], tab, bs, 1)[::3] == ([[0, 0, 0, -1]], 4)


# ---- waits ---------------------------------------------------------------------------------------
def _attention(hd, spans, nh=8, nkv=2, bs=32):
    """(q, cache, tables, row_seq, row_ctx): random codes; spans lists (context before, rows) of each sequence."""
    g = torch.Generator(device=DEV).manual_seed(hd)
    need = [-(-(a + n) // bs) for a, n in spans]
    cache = torch.randint(0, 256, kv4.cache_shape(sum(need), nkv, bs, hd), dtype=torch.uint8, device=DEV, generator=g)
    pairs = torch.rand(*cache.shape[:3], 64 * (hd // 64), device=DEV, generator=g) * 0.2 + 0.05
    cache[..., 16 * hd:] = pairs.half().view(torch.uint8)
    tab, at = torch.zeros(len(spans), max(need), dtype=torch.int32, device=DEV), 0
    for i, m in enumerate(need):
        tab[i, :m] = torch.arange(at, at + m, device=DEV)
        at += m
    row_seq = _ints([i for i, (_, n) in enumerate(spans) for _ in range(n)])
    row_ctx = _ints([a + j + 1 for a, n in spans for j in range(n)])
    q = torch.randn(len(row_seq), nh, hd, device=DEV, generator=g).bfloat16()
    return q, cache, tab, row_seq, row_ctx


WAITING = [(kv4.attention_decode, 64, [(9000, 1), (3, 1), (700, 1)]), (kv4.attention_decode, 128, [(300, 20), (40000, 2)]),
           (kv4.attention_decode, 256, [(20000, 1), (500, 1)]), (kv4.attention_prefill, 64, [(5000, 300), (0, 70)]),
           (kv4.attention_prefill, 128, [(6000, 40)]), (kv4.attention_prefill, 128, [(0, 3000), (100, 1000)])]


def _attend(fn, case, ws):
    out = torch.full((case[0].shape[0], 8 * case[0].shape[2]), 7.0, dtype=torch.bfloat16, device=DEV)
    fn(*case, 0.1, ws, out_bf16=out)
    torch.cuda.synchronize()
    return out


@pytest.mark.parametrize("fn,hd,spans", WAITING)
def test_a_bad_arguments_code_ends_no_wait(fn, hd, spans):
    """The status word holds a bad argument's code, of an earlier launch or of this one's other rows: a row's
    result is what it is without."""
    q, cache, tab, row_seq, row_ctx = case = _attention(hd, spans)
    ws = kv4.Workspace(DEV)
    want = _attend(fn, case, ws)
    assert ws.status.item() == 0
    ws.status.fill_(4)
    for _ in range(5):
        assert torch.equal(_attend(fn, case, ws), want) and ws.status.item() == 4
    ws.status.zero_()
    bad = row_seq.clone()
    bad[-1] = 77
    for _ in range(5):
        assert torch.equal(_attend(fn, (q, cache, tab, bad, row_ctx), ws)[:-1], want[:-1]) and ws.status.item() == 4


@pytest.mark.parametrize("fn,hd,spans", WAITING)
def test_a_wait_that_runs_out_ends_the_launch(fn, hd, spans):
    """Every wait gives up at once, or after a few polls: the launch returns with the timeout's code, over that of a bad
    argument, and after a reset the workspace works as before."""
    case = _attention(hd, spans)
    ws = kv4.Workspace(DEV)
    want = _attend(fn, case, ws)
    polls = ws.wait_polls
    for n, before in ((0, 0), (0, 4), (1, 0), (2, 0), (5, 0), (20, 0)):
        ws.wait_polls = n
        ws.status.fill_(before)
        _attend(fn, case, ws)
        assert ws.status.item() == 3 if n == 0 else ws.status.item() in (0, 3)
        ws.reset()
        ws.wait_polls = polls
        assert torch.equal(_attend(fn, case, ws), want) and ws.status.item() == 0


# ---- inputs that a kernel must not be given ------------------------------------------------------
def _append_args(R=2, nh=8, nkv=2, hd=64, bs=16):
    return dict(qkv=torch.randn(R, (nh + 2 * nkv) * hd, device=DEV), pos=_ints(list(range(R))), slots=_ints(list(range(R))),
                rope=torch.randn(R, hd // 2, 2, device=DEV), rot=hd, style=0,
                q=torch.empty(R, nh, hd, dtype=torch.bfloat16, device=DEV),
                cache=torch.zeros(kv4.cache_shape(2, nkv, bs, hd), dtype=torch.uint8, device=DEV), nh=nh, nkv=nkv, hd=hd)


def test_append_refuses_a_rotation_table_off_its_boundary():
    """(cos, sin) pairs are read as 8 bytes."""
    a = _append_args()
    n = a["rope"].numel()
    shifted = torch.zeros(n + 2, device=DEV)
    a["rope"] = shifted[1:n + 1].view(2, 32, 2)
    with pytest.raises(RuntimeError, match="8-byte aligned"):
        kv4.rope_append(*a.values())
    a["rope"] = shifted[2:].view(2, 32, 2)
    kv4.rope_append(*a.values())
    torch.cuda.synchronize()


@pytest.mark.parametrize("shape", [(2, 0, 1), (2, 2, 0), (0, 0, 0)])
def test_a_cache_without_heads_or_tokens_is_refused(shape):
    """The host divides by the kv heads, the kernels by the block size."""
    cache = torch.zeros(*shape, 18 * 64, dtype=torch.uint8, device=DEV)
    ws, one = kv4.Workspace(DEV), _ints([0])
    q, out = (torch.zeros(*s, dtype=torch.bfloat16, device=DEV) for s in ((1, 4, 64), (1, 256)))
    for fn in (kv4.attention_decode, kv4.attention_prefill):
        with pytest.raises(RuntimeError, match="kv heads and a block size"):
            fn(q, cache, _ints([[0]]), one, one, 0.1, ws, out_bf16=out)
    with pytest.raises(RuntimeError, match="kv heads and a block size"):
        kv4.gather(cache, one, torch.zeros(1, shape[1], 64, dtype=torch.bfloat16, device=DEV), None)
    a = _append_args(R=1)
    a["cache"] = cache
    with pytest.raises(RuntimeError, match="kv heads and a block size"):
        kv4.rope_append(*a.values())
    # blocks alone may be none: every slot is past such a cache
    none = torch.zeros(kv4.cache_shape(0, 2, 16, 64), dtype=torch.uint8, device=DEV)
    k = torch.ones(1, 2, 64, dtype=torch.bfloat16, device=DEV)
    kv4.gather(none, one, k, None)
    assert (k == 0).all()


def test_outputs_whose_rows_lie_over_one_another_are_refused():
    q, cache, tab, row_seq, row_ctx = _attention(64, [(5, 3)])
    ws = kv4.Workspace(DEV)
    for fn in (kv4.attention_decode, kv4.attention_prefill):
        for dtype, name in ((torch.bfloat16, "out_bf16"), (torch.float32, "out")):
            one = torch.zeros(1, 512, dtype=dtype, device=DEV)
            with pytest.raises(RuntimeError, match="over one another"):
                fn(q, cache, tab, row_seq, row_ctx, 0.1, ws, **{name: one.expand(3, 512)})
            with pytest.raises(RuntimeError, match="over one another"):
                fn(q, cache, tab, row_seq, row_ctx, 0.1, ws, **{name: one.new_zeros(2048).as_strided((3, 512), (504, 1))})
    a = _append_args()
    a["q"] = a["q"][:1].expand(2, 8, 64)
    with pytest.raises(RuntimeError, match="over one another"):
        kv4.rope_append(*a.values())


# ---- sinks that are not finite -------------------------------------------------------------------
@pytest.mark.parametrize("fn", [kv4.attention_decode, kv4.attention_prefill])
@pytest.mark.parametrize("spans", [[(40, 1)], [(9000, 1)], [(9000, 3), (0, 300), (77, 1)]])
def test_sinks_that_are_not_finite(fn, spans):
    """However a row's keys are divided up: a NaN sink gives NaN, one of +infinity takes all the weight, one of
    -infinity none, and the other heads do not notice."""
    case = _attention(64, spans)
    ws, nan, inf = kv4.Workspace(DEV), float("nan"), float("inf")
    sinks = torch.tensor([0.5, nan, inf, -inf, 3e38, -3e38, 2.0, -1.0], device=DEV)
    out = []
    for s in (sinks, torch.where(sinks.isfinite() & (sinks.abs() < 9), sinks, 0.0), None):
        o = torch.zeros(case[0].shape[0], 8, 64, device=DEV)
        fn(*case, 0.1, ws, out=o.view(-1, 512), sinks=s)
        out.append(o)
    got, finite, plain = out
    assert got[:, 1].isnan().all() and not got[:, [0, 2, 3, 4, 5, 6, 7]].isnan().any()
    assert (got[:, [2, 4]].abs() < 1e-30).all()
    assert torch.equal(got[:, [0, 6, 7]], finite[:, [0, 6, 7]])
    assert torch.allclose(got[:, [3, 5]], plain[:, [3, 5]], rtol=1e-6, atol=0)  # a sum of one term more
    assert ws.status.item() == 0
