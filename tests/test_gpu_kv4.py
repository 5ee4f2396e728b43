"""The 4-bit paged KV cache (ops/kv4.py) against plain implementations in 64 bits.

The oracle reads the cache code by code from the documented byte positions, so it shares nothing
with the kernels' fragment-order reads. Tolerances follow from the roundings a kernel may make:
float16 softmax weights, keys and values (2^-11 relative each) and the output's own type."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from hawking_b200.ops import kv4  # noqa: E402

DEV = "cuda"
LAYOUTS = [(32, 8, 128), (8, 2, 64), (16, 2, 256), (6, 2, 128), (16, 1, 64), (5, 5, 128), (16, 1, 256), (14, 2, 64)]


# ---- the format, element by element ----------------------------------------------------------------
def _positions(hd):
    """Byte and nibble of every (token of a unit, head dim), keys and values."""
    t, d = torch.arange(16)[:, None], torch.arange(hd)[None]
    row = min(hd, 128) // 2
    r, nib = d % 128, (d % 8) // 2 + 4 * (d % 2)
    kb = (d // 128) * 16 * row + t * row + ((r // 8) % 4) * (row // 4) + (r // 32) * 4 + nib // 2
    kn = (nib % 2).expand_as(kb)
    r, nib = d % 64, (d % 4) + 4 * (t % 2)
    vb = 8 * hd + (d // 64) * 512 + ((r % 32) // 4) * 64 + ((t % 8) // 2) * 16 + (r // 32) * 8 + (t // 8) * 4 + nib // 2
    return kb, kn, vb, (nib % 2).expand_as(vb)


def _values(cache, hd):
    """float64 keys and values [blocks, kv_heads, block_size, hd] of a whole cache (on its device)."""
    kb, kn, vb, vn = (x.to(cache.device) for x in _positions(hd))
    n = cache.shape[:3]

    def codes(b, o):
        raw = cache[..., b.reshape(-1)].long().reshape(*n, 16, hd)
        return torch.where(o.bool(), raw >> 4, raw & 15).double()

    pairs = cache[..., 16 * hd:].contiguous().view(torch.float16).double().reshape(*n, 2, 16, hd // 64, 2)
    out = []
    for i, c in enumerate((codes(kb, kn), codes(vb, vn))):
        p = pairs[..., i, :, :, :].repeat_interleave(64, dim=-2)
        out.append((p[..., 1] + p[..., 0] * (c - 8)).reshape(n[0], n[1], n[2] * 16, hd))
    return out


def _random_cache(g, blocks, nkv, bs, hd):
    cache = torch.randint(0, 256, kv4.cache_shape(blocks, nkv, bs, hd), dtype=torch.uint8, device=DEV, generator=g)
    n = 32 * (hd // 64)
    s = torch.rand(*cache.shape[:3], n, device=DEV, generator=g) * 0.2 + 0.05
    c = torch.randn(*cache.shape[:3], n, device=DEV, generator=g) * 0.2
    cache[..., 16 * hd:] = torch.stack([s, c], -1).half().reshape(*cache.shape[:3], 2 * n).view(torch.uint8)
    return cache


def _attention_case(seed, nh, nkv, hd, bs, spans, stale=True):
    """spans: [(context before, rows)] per sequence. Every cache byte that no row may see is 0xff, which
    reads as NaN pairs."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    need = [max(1, -(-(a + n) // bs)) for a, n in spans]
    blocks = sum(need) + 2
    cache = _random_cache(g, blocks, nkv, bs, hd)
    perm = torch.randperm(blocks, device=DEV, generator=g).int()
    tab = torch.full((len(spans) + 1, max(need) + 1), 0, dtype=torch.int32, device=DEV)
    row_seq, row_ctx, at = [], [], 0
    if stale:
        keep = cache.clone()
        cache.fill_(255)
    for i, ((a, n), m) in enumerate(zip(spans, need)):
        tab[i, :m] = perm[at:at + m]
        if stale:
            for t in range(0, a + n, 16):
                b, u = int(perm[at + t // bs]), t % bs // 16
                cache[b, :, u] = keep[b, :, u]
                if a + n - t < 16:  # tokens past the end: NaN pairs
                    live = a + n - t
                    pairs = cache[b, :, u, 16 * hd:].reshape(nkv, 2, 16, -1)
                    pairs[:, :, live:] = 255
        row_seq += [i] * n
        row_ctx += [a + j + 1 for j in range(n)]
        at += m
    q = (torch.randn(len(row_seq), nh, hd, device=DEV, generator=g) * 2).bfloat16()
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    return q, cache, tab, ints(row_seq), ints(row_ctx)


def _attention64(q, cache, tab, row_seq, row_ctx, scale, sinks=None):
    """(output, bound on the error that rounding k, v and the weights to float16 makes), float64."""
    R, nh, hd = q.shape
    bs, nkv = cache.shape[2] * 16, cache.shape[1]
    out = torch.zeros(R, nh, hd, dtype=torch.float64, device=DEV)
    tol = torch.zeros(R, nh, 1, dtype=torch.float64, device=DEV)
    seqs = row_seq.tolist()
    for seq in sorted(set(seqs)):
        rows = torch.tensor([i for i, s in enumerate(seqs) if s == seq], device=DEV)
        ctx = row_ctx[rows].long()
        n = int(ctx.max())
        if n <= 0:
            continue
        k, v = _values(cache[tab[seq, : -(-n // bs)].long()], hd)
        k, v = (x.permute(0, 2, 1, 3).reshape(-1, nkv, hd)[:n] for x in (k, v))
        seen = torch.arange(n, device=DEV)[None] < ctx[:, None]
        G = nh // nkv
        for h in range(nh):
            # rows of this sequence see different lengths: unseen keys may hold NaN
            kk = torch.where(torch.isnan(k[:, h // G]), 0.0, k[:, h // G])
            vv = torch.where(torch.isnan(v[:, h // G]), 0.0, v[:, h // G])
            qq = q[rows, h].double()
            s = (qq @ kk.T * scale).masked_fill(~seen, -math.inf)
            if sinks is not None:
                s = torch.cat([s, sinks[h].double().expand(len(rows), 1)], 1)
            w = torch.nan_to_num(torch.softmax(s, -1))[:, :n]
            out[rows, h] = w @ vv
            shift = (qq.abs() @ kk.abs().T * scale * 2.0 ** -11).masked_fill(~seen, 0).amax(-1)
            tol[rows, h, 0] = vv.abs().amax() * (2.0 ** -10 + 2 * shift + 1e-5)
    return out.reshape(R, nh * hd), tol.expand(R, nh, hd).reshape(R, nh * hd)


def _check(out, ref, tol, bf16):
    o = out.double()
    assert torch.isfinite(o).all()
    assert ((o - ref).abs() <= tol + (2.0 ** -8 * ref.abs() if bf16 else 0) + 1e-6).all(), (o - ref).abs().max()
    norm = ref.norm()
    if norm > 0:  # random roundings: 2^-11 / sqrt 3 each of k, v, weights; 2^-8 / sqrt 3 of a bf16 output
        assert (o - ref).norm() <= (4e-3 if bf16 else 1.5e-3) * norm


def _run(fn, q, cache, tab, row_seq, row_ctx, sinks=None, bf16=True):
    ws = kv4.Workspace(DEV)
    R, nh, hd = q.shape
    out = torch.full((R, nh * hd), float("nan"), dtype=torch.bfloat16 if bf16 else torch.float32, device=DEV)
    fn(q, cache, tab, row_seq, row_ctx, 1 / math.sqrt(hd), ws, sinks=sinks, **{"out_bf16" if bf16 else "out": out})
    torch.cuda.synchronize()
    assert ws.status.item() == 0
    return out


# ---- attention -------------------------------------------------------------------------------------
@pytest.mark.parametrize("nh,nkv,hd", LAYOUTS)
@pytest.mark.parametrize("bs", [16, 64, 48])
def test_decode_matches_64bit(nh, nkv, hd, bs):
    ctxs = [1, 2, 15, 16, 17, 63, 64, 65, 127, 129, 500, 1333]
    case = _attention_case(hd + nh + bs, nh, nkv, hd, bs, [(c - 1, 1) for c in ctxs])
    ref, tol = _attention64(*case, 1 / math.sqrt(hd))
    _check(_run(kv4.attention_decode, *case), ref, tol, True)
    _check(_run(kv4.attention_decode, *case, bf16=False), ref, tol, False)


@pytest.mark.parametrize("rows,ctx", [(1, 1), (1, 5000), (2, 20011), (70, 300), (300, 33)])
def test_decode_row_counts(rows, ctx):
    spans = [(max(0, ctx - 1 - 7 * (i % 5)), 1) for i in range(rows)]
    case = _attention_case(rows, 16, 4, 128, 64, spans)
    ref, tol = _attention64(*case, 1 / math.sqrt(128))
    _check(_run(kv4.attention_decode, *case), ref, tol, True)


@pytest.mark.parametrize("rows,columns", [(600, 4), (40, 1 << 22)])
def test_decode_in_several_launches(rows, columns):
    """More rows than a launch holds, and a table so wide that a launch's work is bounded by what it could hold."""
    q, cache, tab, row_seq, row_ctx = _attention_case(rows, 16, 8, 64, 16, [(i % 40, 1) for i in range(rows)])
    wide = torch.full((tab.shape[0], columns), 1 << 30, dtype=torch.int32, device=DEV)
    wide[:, :tab.shape[1]] = tab
    case = (q, cache, wide, row_seq, row_ctx)
    ref, tol = _attention64(*case, 1 / math.sqrt(64))
    _check(_run(kv4.attention_decode, *case), ref, tol, True)


@pytest.mark.parametrize("fn", [kv4.attention_decode, kv4.attention_prefill])
def test_attention_empty_rows_and_sinks(fn):
    q, cache, tab, row_seq, row_ctx = _attention_case(3, 8, 2, 128, 32, [(70, 4), (0, 3), (200, 2)])
    row_ctx[1] = 0       # a masked row inside a run
    row_ctx[5] = 0
    row_ctx[8] = -3      # negative reads as none
    sinks = torch.tensor([0.5, -2.0, 3.0, 0.0, 1.0, -30.0, 8.0, 0.1], device=DEV)
    for s in (None, sinks):
        ref, tol = _attention64(q, cache, tab, row_seq, row_ctx, 1 / math.sqrt(128), s)
        out = _run(fn, q, cache, tab, row_seq, row_ctx, sinks=s)
        assert (out[[1, 5, 8]] == 0).all()
        _check(out, ref, tol, True)


@pytest.mark.parametrize("nh,nkv,hd", [l for l in LAYOUTS if l[2] <= 128])
@pytest.mark.parametrize("bs", [16, 64, 48])
def test_prefill_matches_64bit(nh, nkv, hd, bs):
    spans = [(0, 1), (0, 130), (517, 70), (3, 2), (100, 33)]
    case = _attention_case(hd + nh + bs, nh, nkv, hd, bs, spans)
    ref, tol = _attention64(*case, 1 / math.sqrt(hd))
    _check(_run(kv4.attention_prefill, *case), ref, tol, True)
    _check(_run(kv4.attention_prefill, *case, bf16=False), ref, tol, False)


@pytest.mark.parametrize("past,rows", [(0, 1), (0, 700), (3000, 1), (5000, 40), (1111, 257)])
def test_prefill_one_sequence(past, rows):
    case = _attention_case(past + rows, 16, 4, 128, 64, [(past, rows)])
    ref, tol = _attention64(*case, 1 / math.sqrt(128))
    _check(_run(kv4.attention_prefill, *case), ref, tol, True)


@pytest.mark.parametrize("fn", [kv4.attention_decode, kv4.attention_prefill])
def test_attention_extreme_scores_and_scales(fn):
    """Large and tiny scales, zero scales and scores far apart: no overflow, no NaN."""
    hd = 128
    q, cache, tab, row_seq, row_ctx = _attention_case(9, 8, 2, hd, 32, [(300, 3), (90, 2)], stale=False)
    p = cache[..., 16 * hd:].view(torch.float16).reshape(*cache.shape[:3], 2, 16, hd // 64, 2)
    p[:, :, :, 1, 0:4, :, :] = torch.tensor([4000.0, 12000.0], device=DEV).half()   # huge values
    p[:, :, :, 1, 4:8, :, 0] = 0                                                   # constant groups
    p[:, :, :, 1, 8:12, :, 0] = 3e-6                                               # subnormal scales
    p[:, :, :, 0, 5, :, 1] = 100.0                                                 # one dominant key per unit
    ref, tol = _attention64(q, cache, tab, row_seq, row_ctx, 1 / math.sqrt(hd))
    out = _run(fn, q, cache, tab, row_seq, row_ctx)
    assert ((out.double() - ref).abs() <= tol + 2.0 ** -8 * ref.abs() + 1e-6).all()


@pytest.mark.parametrize("fn", [kv4.attention_decode, kv4.attention_prefill])
def test_attention_nan_group_reaches_only_rows_that_see_it(fn):
    hd = 64
    q, cache, tab, row_seq, row_ctx = _attention_case(4, 4, 2, hd, 16, [(20, 30)], stale=False)
    blk, off = int(tab[0, 40 // 16]), 40 % 16
    cache[blk, 0, 0].view(torch.float16)[8 * hd + (16 + off) * 2] = float("nan")  # value scale of token 40, head 0
    ws = kv4.Workspace(DEV)
    out = torch.empty(30, 4 * hd, device=DEV)
    fn(q, cache, tab, row_seq, row_ctx, 0.125, ws, out=out)
    sees = (row_ctx > 40)[:, None].expand(-1, 2 * hd)
    assert torch.isnan(out[:, : 2 * hd][sees]).all() and torch.isfinite(out[:, : 2 * hd][~sees]).all()
    assert torch.isfinite(out[:, 2 * hd:]).all()


@pytest.mark.parametrize("fn", [kv4.attention_decode, kv4.attention_prefill])
def test_attention_strided_rows_and_other_stream(fn):
    q, cache, tab, row_seq, row_ctx = _attention_case(6, 8, 2, 64, 32, [(100, 20), (31, 5)])
    R = q.shape[0]
    wide = torch.zeros(R, 12, 64, dtype=torch.bfloat16, device=DEV)
    wide[:, 2:10] = q
    outw = torch.full((R, 1024), 7.0, dtype=torch.bfloat16, device=DEV)
    ref, tol = _attention64(q, cache, tab, row_seq, row_ctx, 0.125)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ws = kv4.Workspace(DEV)
        fn(wide[:, 2:10], cache, tab, row_seq, row_ctx, 0.125, ws, out_bf16=outw[:, 256:768])
    s.synchronize()
    _check(outw[:, 256:768], ref, tol, True)
    assert (outw[:, :256] == 7).all() and (outw[:, 768:] == 7).all()


@pytest.mark.parametrize("fn", [kv4.attention_decode, kv4.attention_prefill])
def test_attention_repeats_bitwise_and_in_a_graph(fn):
    q, cache, tab, row_seq, row_ctx = _attention_case(8, 32, 8, 128, 64, [(4000, 9), (600, 1), (0, 40)])
    ws = kv4.Workspace(DEV)
    out = torch.zeros(50, 32 * 128, dtype=torch.bfloat16, device=DEV)
    call = lambda: fn(q, cache, tab, row_seq, row_ctx, 0.1, ws, out_bf16=out)  # noqa: E731
    call()
    first = out.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    for _ in range(20):
        out.zero_()
        g.replay()
        assert torch.equal(out, first)


@pytest.mark.parametrize("fn", [kv4.attention_decode, kv4.attention_prefill])
def test_attention_bad_indices_set_the_status(fn):
    q, cache, tab, row_seq, row_ctx = _attention_case(5, 8, 2, 64, 32, [(100, 4), (40, 4)])
    ref = _run(fn, q, cache, tab, row_seq, row_ctx)
    for what in ("seq", "block"):
        ws, rs, tb = kv4.Workspace(DEV), row_seq.clone(), tab.clone()
        if what == "seq":
            rs[4:] = 99
        else:
            tb[1, 0] = cache.shape[0] + 7
        out = torch.empty(8, 512, dtype=torch.bfloat16, device=DEV)
        fn(q, cache, tb, rs, row_ctx, 0.125, ws, out_bf16=out)
        assert ws.status.item() == 4
        assert torch.equal(out[:4], ref[:4])
        assert torch.isfinite(out).all()


def test_attention_and_gather_past_4_gib():
    """Byte offsets beyond 32 bits: the sequence's blocks lie at the end of a 4.6 GB cache."""
    hd, nkv, bs = 128, 8, 64
    blocks = (4_600_000_000 // (nkv * bs // 16 * 18 * hd))
    cache = torch.empty(kv4.cache_shape(blocks, nkv, bs, hd), dtype=torch.uint8, device=DEV)
    small = _attention_case(2, 32, nkv, hd, bs, [(150, 9)], stale=False)
    q, c, tab, row_seq, row_ctx = small
    cache[-c.shape[0]:] = c
    far = tab + (blocks - c.shape[0])
    for fn in (kv4.attention_decode, kv4.attention_prefill):
        assert torch.equal(_run(fn, q, cache, far, row_seq, row_ctx), _run(fn, *small))
    slots = (far[0, :2].long()[:, None] * bs + torch.arange(bs, device=DEV)).reshape(-1).int()
    k, v = (torch.empty(128, nkv, hd, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    kv4.gather(cache, slots, k, v)
    rk, rv = _values(c[tab[0, :2].long()], hd)
    assert torch.equal(k, rk.permute(0, 2, 1, 3).reshape(128, nkv, hd).float().bfloat16())
    assert torch.equal(v, rv.permute(0, 2, 1, 3).reshape(128, nkv, hd).float().bfloat16())


# ---- append and gather -----------------------------------------------------------------------------
def _rope(n, rot, theta=10000.0):
    i = torch.arange(rot // 2, dtype=torch.float64)
    ang = torch.arange(n, dtype=torch.float64)[:, None] * theta ** (-2.0 * i / max(rot, 1))
    return torch.stack([torch.cos(ang), torch.sin(ang)], -1).float().to(DEV)


def _pack_pairs(x):
    """The documented quantiser in fp32: (values that the codes stand for, s, c), float64."""
    g = x.float().reshape(*x.shape[:-1], -1, 64).clamp(-65024, 65024)
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    s = ((hi - lo) * torch.full_like(hi, 1.0 / 15.0)).half().float()
    c = (lo + 8.0 * s).half().float()
    code = torch.where(s > 0, torch.round((g - c) / s) + 8, torch.full_like(g, 8)).clamp(0, 15)
    return (c.double() + s.double() * (code.double() - 8)).reshape(x.shape), s.double(), c.double()


def _rotate(x, rope, style, dtype):
    x = x.to(dtype).clone()
    rot = rope.shape[1] * 2
    cs, sn = rope[:, None, :, 0].to(dtype), rope[:, None, :, 1].to(dtype)
    ia = torch.arange(rot // 2, device=DEV) * (2 if style == 0 else 1)
    ib = ia + (1 if style == 0 else rot // 2)
    a, b = x[..., ia], x[..., ib]
    x[..., ia], x[..., ib] = a * cs - b * sn, a * sn + b * cs
    return x


@pytest.mark.parametrize("nh,nkv,hd", [(32, 8, 128), (8, 2, 64), (7, 1, 64), (16, 2, 256), (3, 3, 128)])
@pytest.mark.parametrize("style,part", [(0, 1), (1, 1), (0, 2), (1, 4), (1, 3)])
def test_append_values_exact(nh, nkv, hd, style, part):
    """Without norms every operation of the append is defined to the last bit."""
    g = torch.Generator(device=DEV).manual_seed(nh + hd + style + part)
    rot = hd // part // 2 * 2 if part != 3 else hd // 4 + 2
    R, bs, blocks = 37, 32, 7
    qkv = torch.randn(R, (nh + 2 * nkv) * hd, device=DEV, generator=g)
    bias = torch.randn((nh + 2 * nkv) * hd, device=DEV, generator=g)
    rope = _rope(500, rot)
    pos = torch.randint(0, 500, (R,), device=DEV, generator=g).int()
    slots = torch.randperm(blocks * bs, device=DEV, generator=g)[:R].int()
    cache = torch.zeros(kv4.cache_shape(blocks, nkv, bs, hd), dtype=torch.uint8, device=DEV)
    q = torch.empty(R, nh, hd, dtype=torch.bfloat16, device=DEV)
    kv4.rope_append(qkv, pos, slots, rope, rot, style, q, cache, nh, nkv, hd, bias=bias)
    x = (qkv + bias).reshape(R, -1, hd)
    turned = _rotate(x[:, :nh + nkv], rope[pos.long()], style, torch.float32)
    assert torch.equal(q, turned[:, :nh].bfloat16())
    k, v = _values(cache, hd)
    s = slots.long()
    for got, want in ((k, turned[:, nh:]), (v, x[:, nh + nkv:])):
        assert torch.equal(got[s // bs, :, s % bs], _pack_pairs(want)[0])
    # nothing else was written
    rest = torch.ones(blocks * bs, dtype=torch.bool, device=DEV)
    rest[s] = False
    rest = rest.reshape(blocks, bs)
    assert (k.permute(0, 2, 1, 3)[rest] == 0).all() and (v.permute(0, 2, 1, 3)[rest] == 0).all()


@pytest.mark.parametrize("rows,nh,nkv,hd", [(700, 32, 8, 128), (1500, 8, 3, 64), (2200, 7, 1, 64), (1000, 16, 2, 256)])
@pytest.mark.parametrize("style,part", [(0, 1), (1, 1), (1, 2)])
@pytest.mark.parametrize("bias", [False, True])
def test_append_many_rows_exact(rows, nh, nkv, hd, style, part, bias):
    """Several heads per warp, and codes half way between two integers."""
    g = torch.Generator(device=DEV).manual_seed(rows + style)
    bs, rot = 16, hd // part
    blocks = -(-rows // bs)
    x = torch.randn(rows, nh + 2 * nkv, hd, device=DEV, generator=g)
    x[:, nh + nkv:] = torch.randint(0, 31, (rows, nkv, hd), device=DEV, generator=g) / 2
    b = torch.randint(-3, 4, ((nh + 2 * nkv) * hd,), device=DEV, generator=g).float() if bias else None
    rope, pos = _rope(rows, rot), torch.arange(rows, dtype=torch.int32, device=DEV)
    slots = torch.randperm(blocks * bs, device=DEV, generator=g)[:rows].int()
    cache = torch.zeros(kv4.cache_shape(blocks, nkv, bs, hd), dtype=torch.uint8, device=DEV)
    q = torch.empty(rows, nh, hd, dtype=torch.bfloat16, device=DEV)
    kv4.rope_append(x.reshape(rows, -1), pos, slots, rope, rot, style, q, cache, nh, nkv, hd, bias=b)
    if bias:
        x = x + b.reshape(-1, hd)
    turned = _rotate(x[:, :nh + nkv], rope, style, torch.float32)
    assert torch.equal(q, turned[:, :nh].bfloat16())
    s = slots.long()
    for got, want in zip(_values(cache, hd), (turned[:, nh:], x[:, nh + nkv:])):
        assert torch.equal(got[s // bs, :, s % bs], _pack_pairs(want)[0])


@pytest.mark.parametrize("hd,rot,style", [(64, 64, 0), (128, 128, 1), (256, 64, 1)])
def test_append_norm_against_64bit(hd, rot, style):
    g = torch.Generator(device=DEV).manual_seed(hd)
    R, nh, nkv, bs = 50, 6, 2, 16
    qkv = torch.randn(R, (nh + 2 * nkv) * hd, device=DEV, generator=g) * 3
    qn, kn = (1 + 0.2 * torch.randn(hd, device=DEV, generator=g) for _ in range(2))
    rope, pos = _rope(64, rot), torch.arange(R, device=DEV, dtype=torch.int32)
    tab = torch.tensor([[9, 9, 9, 9], [3, 0, 2, 1]], dtype=torch.int32, device=DEV)
    cache = torch.zeros(kv4.cache_shape(4, nkv, bs, hd), dtype=torch.uint8, device=DEV)
    q = torch.empty(R, nh, hd, dtype=torch.bfloat16, device=DEV)
    kv4.rope_append(qkv, pos, None, rope, rot, style, q, cache, nh, nkv, hd, q_norm=qn, k_norm=kn, eps=1e-5,
                    block_tables=tab, row_seq=torch.ones(R, dtype=torch.int32, device=DEV))
    x = qkv.double().reshape(R, -1, hd)
    x = torch.cat([x[:, :nh + nkv] / (x[:, :nh + nkv].pow(2).mean(-1, keepdim=True) + 1e-5).sqrt(), x[:, nh + nkv:]], 1)
    x[:, :nh] *= qn.double()
    x[:, nh:nh + nkv] *= kn.double()
    turned = _rotate(x[:, :nh + nkv], rope[pos.long()], style, torch.float64)
    # bf16 rounding, and a few fp32 roundings of values of at most |x| of both partners
    assert ((q.double() - turned[:, :nh]).abs() <= 2.0 ** -8 * turned[:, :nh].abs() + 1e-5).all()
    k, v = _values(cache, hd)
    k, v = (t[[3, 0, 2, 1]].permute(0, 2, 1, 3).reshape(64, nkv, hd)[:R] for t in (k, v))
    for got, want in ((k, turned[:, nh:]), (v, x[:, nh + nkv:])):
        _, s, c = _pack_pairs(want)
        # half a step; the ends of the range give by the float16 rounding of s and c
        tol = (0.5 * s + 2.0 ** -11 * (c.abs() + 16 * s) + 1e-5).expand(R, nkv, hd // 64, 64).reshape(R, nkv, hd)
        assert ((got - want).abs() <= tol).all()


def test_append_odd_values_and_skipped_rows():
    hd, nh, nkv, bs = 128, 2, 1, 16
    R = 10
    qkv = torch.zeros(R, (nh + 2 * nkv) * hd, device=DEV)
    kv = qkv[:, nh * hd:]
    kv[0, :] = 1.25                      # constant groups
    kv[1, 3], kv[1, 70] = float("nan"), float("inf")
    kv[2, 0], kv[2, 1] = 1e30, -1e30     # clamped
    kv[3, :64] = torch.linspace(-1e-6, 1e-6, 64, device=DEV)
    kv[4, 0] = 3.4e38
    pos = torch.zeros(R, dtype=torch.int32, device=DEV)
    pos[8], pos[9] = 5, -1               # outside the table of 5 rows: left alone
    slots = torch.arange(R, dtype=torch.int32, device=DEV)
    slots[5], slots[6], slots[7] = -1, 32, 10 ** 6  # no slot, past the cache
    kv[5:] = 9.0
    cache = torch.zeros(kv4.cache_shape(2, nkv, bs, hd), dtype=torch.uint8, device=DEV)
    q = torch.full((R, nh, hd), 3.0, dtype=torch.bfloat16, device=DEV)
    rope = torch.zeros(5, hd // 2, 2, device=DEV)
    rope[..., 0] = 1.0
    kv4.rope_append(qkv, pos, slots, rope, hd, 0, q, cache, nh, nkv, hd)
    k, v = _values(cache, hd)
    k = k[0, 0]
    assert (k[0] == 1.25).all() and (v[0, 0, 0] == 1.25).all()
    assert torch.isnan(k[1]).all()       # one odd value in each of the two groups
    assert (v[0, 0, 1] == 0).all()
    assert torch.isfinite(k[2]).all() and k[2, 0] > 60000 and k[2, 1] < -60000
    assert torch.equal(k[3, :64], _pack_pairs(kv[3, :64])[0])  # a subnormal scale
    assert torch.isfinite(k[4]).all() and k[4, 0] > 60000
    assert (k[5:] == 0).all() and (cache[1] == 0).all()
    assert (q[:8] == 0).all() and (q[8:] == 3).all()


@pytest.mark.parametrize("nkv,hd,bs", [(8, 128, 64), (2, 64, 16), (2, 256, 48), (1, 128, 32)])
def test_gather_exact(nkv, hd, bs):
    g = torch.Generator(device=DEV).manual_seed(bs)
    cache = _random_cache(g, 9, nkv, bs, hd)
    k, v = _values(cache, hd)
    for slots in (torch.arange(9 * bs), torch.randperm(9 * bs)[:101], torch.tensor([5]), torch.arange(3, 3 + 4 * bs),
                  torch.tensor([0, -1, 9 * bs, 2 ** 31 - 1, 7])):
        s = slots.to(DEV)
        ok = (s >= 0) & (s < 9 * bs)
        t = torch.where(ok, s, 0)
        ko, vo = (torch.full((len(s), nkv, hd), 5.0, dtype=torch.bfloat16, device=DEV) for _ in range(2))
        kv4.gather(cache, s.int(), ko, vo)
        for got, want in ((ko, k), (vo, v)):
            want = want[t // bs, :, t % bs].float().bfloat16() * ok[:, None, None]
            assert torch.equal(got, want)
        only = torch.zeros_like(vo)
        kv4.gather(cache, s.int(), None, only)
        assert torch.equal(only, vo)


# ---- rows of a step --------------------------------------------------------------------------------
def _plan_ref(seq, cached, new, tab, bs, cap, free):
    tab, used, rows = tab.copy(), 0, []
    for q, a, n in zip(seq, cached, new):
        for col in range(-(-a // bs), -(-(a + n) // bs) if n else 0):
            tab[q, col] = free[used]
            used += 1
        rows += [(p, q, p + 1, tab[q, p // bs] * bs + p % bs) for p in range(a, a + n)]
    rows += [(0, 0, 0, -1)] * (cap - len(rows))
    return rows, tab, used


def _plan(seq, cached, new, tab, bs, cap, free=None):
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    out = torch.full((4, cap), 77, dtype=torch.int32, device=DEV)
    t, taken, status = ints(tab), ints([-5]), ints([0])
    kv4.plan_rows(ints(seq), ints(cached), ints(new), t, bs, *out.unbind(0),
                  free_blocks=None if free is None else ints(free), taken=taken, status=status)
    torch.cuda.synchronize()
    return out.t().tolist(), t.cpu().numpy(), taken.item(), status.item()


@pytest.mark.parametrize("S,bs,top,new_top", [(1, 16, 40, 1), (3, 64, 200, 90), (64, 16, 300, 1), (600, 32, 500, 3),
                                             (33, 48, 100, 700), (2000, 16, 60, 2)])
def test_plan_matches_reference(S, bs, top, new_top):
    import numpy as np
    r = np.random.RandomState(S)
    cached, new = r.randint(0, top, S), r.randint(0, new_top + 1, S)
    cached[0] = 0
    seq = r.permutation(S + 5)[:S]
    width = -(-(top + new_top) // bs) + 1
    have = -(-cached // bs)
    perm = r.permutation(int(have.sum()) + S * (width + 1))
    tab, at = np.zeros((S + 5, width), np.int32), 0
    for q, n in zip(seq, have):
        tab[q, :n] = perm[at:at + n]
        at += n
    cap = int(new.sum()) + 11
    rows, want_tab, used = _plan_ref(seq, cached, new, tab, bs, cap, perm[at:])
    got, got_tab, taken, status = _plan(seq, cached, new, tab, bs, cap, perm[at:])
    assert status == 0 and taken == used
    assert (got_tab == want_tab).all()
    assert got == [list(map(int, x)) for x in rows]
    # the same rows over complete tables, with nothing taken
    got2, tab2, taken2, status2 = _plan(seq, cached, new, want_tab, bs, cap)
    assert got2 == got and (tab2 == want_tab).all() and taken2 == 0 and status2 == 0


def test_plan_refusals_set_the_status():
    tab = [[5, 6, 0], [7, 0, 0]]
    base = dict(seq=[0, 1], cached=[20, 3], new=[2, 1], tab=tab, bs=16, cap=4, free=[9, 8])
    good = [[20, 0, 21, 100], [21, 0, 22, 101], [3, 1, 4, 115], [0, 0, 0, -1]]
    rows, _, taken, status = _plan(**base)
    assert (rows, taken, status) == (good, 0, 0)
    for change in (dict(seq=[0, 2]), dict(seq=[0, -1]), dict(cached=[20, -1]), dict(new=[2, -1]), dict(cached=[20, 48])):
        rows, t, _, status = _plan(**{**base, **change})
        assert status == 4 and rows == good[:2] + [[0, 0, 0, -1]] * 2 and (t == tab).all()
    rows, _, _, status = _plan(**{**base, "cap": 2})     # rows that do not fit are dropped
    assert status == 4 and rows == good[:2]
    # not enough free blocks: the rows without a block have no slot
    rows, t, taken, status = _plan(**{**base, "cached": [32, 16], "free": [9]})
    assert status == 4 and taken == 1 and t.tolist() == [[5, 6, 9], [7, 0, 0]]
    assert rows == [[32, 0, 33, 144], [33, 0, 34, 145], [16, 1, 17, -1], [0, 0, 0, -1]]
    rows, _, taken, status = _plan(**{**base, "cached": [32, 3], "free": []})
    assert status == 4 and taken == 0 and [r[3] for r in rows] == [-1, -1, 115, -1]
    # no requests, no rows
    assert _plan([], [], [], tab, 16, 3)[0] == [[0, 0, 0, -1]] * 3
    assert _plan([], [], [], tab, 16, 0)[3] == 0


def test_refusals():
    ws = kv4.Workspace(DEV)
    q, cache, tab, rs, rc = _attention_case(1, 8, 2, 64, 32, [(10, 2)])
    out = torch.empty(2, 512, dtype=torch.bfloat16, device=DEV)
    bad = [dict(q=q.float()), dict(q=q[:, :7]), dict(q=q[..., :32]), dict(cache=cache[..., :-18]),
           dict(cache=cache[:, :, :1]), dict(cache=cache.cpu()), dict(tab=tab.long()), dict(rs=rs[:1]), dict(rc=rc.long()),
           dict(out=out[:1]), dict(out=out.half()), dict(out=None), dict(tab=tab.t()), dict(out=out[:, 1:])]
    for b in bad:
        a = {**dict(q=q, cache=cache, tab=tab, rs=rs, rc=rc, out=out), **b}
        for fn in (kv4.attention_decode, kv4.attention_prefill):
            with pytest.raises(RuntimeError):
                fn(a["q"], a["cache"], a["tab"], a["rs"], a["rc"], 0.1, ws, out_bf16=a["out"])
    q17 = torch.zeros(2, 34, 64, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(RuntimeError, match="at most 16"):
        kv4.attention_decode(q17, cache, tab, rs, rc, 0.1, ws, out_bf16=torch.empty(2, 34 * 64, dtype=torch.bfloat16,
                                                                                device=DEV))
    c256 = torch.zeros(kv4.cache_shape(2, 2, 32, 256), dtype=torch.uint8, device=DEV)
    with pytest.raises(RuntimeError, match="head_dim 64 or 128"):
        kv4.attention_prefill(torch.zeros(2, 8, 256, dtype=torch.bfloat16, device=DEV), c256, tab, rs, rc, 0.1, ws,
                              out_bf16=torch.empty(2, 2048, dtype=torch.bfloat16, device=DEV))
    qkv = torch.zeros(2, 12 * 64, device=DEV)
    rope = torch.zeros(4, 32, 2, device=DEV)
    ok = dict(qkv=qkv, pos=rs, slots=rs, rope=rope, rot=64, style=0, q=q, cache=cache, nh=8, nkv=2, hd=64)
    kv4.rope_append(*ok.values())
    for b in (dict(qkv=qkv[:, 1:]), dict(qkv=qkv.double()), dict(pos=rs.long()), dict(slots=rs[:1]), dict(rot=63),
              dict(rot=32), dict(style=2), dict(q=q.float()), dict(nkv=1), dict(hd=128), dict(slots=None)):
        with pytest.raises(RuntimeError):
            kv4.rope_append(*{**ok, **b}.values())
    k = torch.empty(2, 2, 64, dtype=torch.bfloat16, device=DEV)
    for a in ((cache, rs.long(), k, k), (cache, rs, k[:1], k), (cache, rs, k.float(), k)):
        with pytest.raises(RuntimeError):
            kv4.gather(*a)
    with pytest.raises(RuntimeError):
        kv4.plan_rows(rs, rs, rs[:1], tab, 16, rs, rs, rs, rs)
    for hd, bs in ((96, 16), (64, 24), (64, 0)):
        with pytest.raises(ValueError):
            kv4.cache_shape(1, 1, bs, hd)
