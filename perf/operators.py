"""The operators of a paged key/value cache held in 4 bits, as measured cases.

A serving step over such a cache lays its rows out on the GPU from the request lengths (``plan``),
rotates the queries and keys and quantises the new keys and values into the cache (``append``),
attends over the cache with one row per sequence (``decode``) or with prompt chunks (``prefill``),
and reads tokens back as 16-bit rows for a snapshot (``gather``).

Cache format. A layer's cache is uint8 [blocks, kv_heads, block_size / 16, 18 * head_dim]: 16 tokens
of one head form a unit of 18 * head_dim bytes. A value is ``c + s * (code - 8)`` with a 4-bit code
and one (s, c) pair of float16 per token and 64 head dims. A unit holds, in order,

* key codes, 32-bit words [head_dim / 128 (at least 1)][token 16][t 4][i] with nibble p + 4 e of a
  word being head dim 128 plane + 32 i + 8 t + 2 p + e (i < 4, or i < 2 for head_dim 64);
* value codes, words [head_dim / 64][g 8][t 4][i 2][h 2] with nibble p + 4 e of a word being token
  8 h + 2 t + e, head dim 64 plane + 32 i + 4 g + p;
* key pairs [token 16][head_dim / 64][s, c], then value pairs of the same shape.

A group is quantised with s = f16((max - min) / 15), c = f16(min + 8 s) and
code = clamp(rint((x - c) / s) + 8, 0, 15) (8 where s is 0).
"""
import math

import numpy as np
import torch

own = False
DEV = "cuda"
_ops = None
_ws = None


def _kv4():
    """The framework's operators and the workspace a program keeps for its stream."""
    global _ops, _ws
    if _ops is None:
        from hawking_b200.ops import kv4
        _ops, _ws = kv4, kv4.Workspace(DEV)
    return _ops, _ws


# ---- cases -------------------------------------------------------------------------------------
# Head layouts are those of this repository's model presets: 32/8 heads of 128 (Llama-3-8B,
# Mixtral), 8/2 of 64 (tiny Llama), 16/2 of 256 (Qwen3-Next's full-attention layers).
def listed():
    return [
        # one decode step of a full batch of 64 requests at mixed lengths: latency
        dict(name="plan-decode-64", op="plan", seqs=64, decode=64, lo=1, hi=8191, chunk_lo=1, chunk_hi=1, bs=64),
        # a continuous-batching step: 448 decoding requests next to 64 prompt chunks of 16 to 1024 tokens
        dict(name="plan-mixed-512", op="plan", seqs=512, decode=448, lo=3, hi=30000, chunk_lo=16, chunk_hi=1024,
             bs=16),
        # decode step of 32 requests on the 256-wide heads: per-head norms, partial rotation by halves
        dict(name="append-decode-32", op="append", rows=32, nh=16, nkv=2, hd=256, rot=64, style=1, norm=True, bs=64,
             pos=4096),
        # a 2048-token prompt chunk, full rotation of adjacent pairs
        dict(name="append-prompt-2048", op="append", rows=2048, nh=32, nkv=8, hd=128, rot=128, style=0, norm=False,
             bs=64, pos=2048),
        # snapshot of one short sequence
        dict(name="gather-777", op="gather", rows=777, nkv=2, hd=64, bs=32, blocks=64),
        # snapshot of a batch of long sequences
        dict(name="gather-65536", op="gather", rows=65536, nkv=8, hd=128, bs=64, blocks=1200),
        # single-user decode at the headline context
        dict(name="decode-1x2048", op="decode", rows=1, nh=32, nkv=8, hd=128, bs=64, lo=2048, hi=2048),
        # a ragged batch of 64: contexts from 200 tokens to the window
        dict(name="decode-64-ragged", op="decode", rows=64, nh=32, nkv=8, hd=128, bs=64, lo=200, hi=8192),
        # two long documents, 256-wide heads in small blocks, odd lengths
        dict(name="decode-2-long", op="decode", rows=2, nh=16, nkv=2, hd=256, bs=16, lo=30001, hi=60001),
        # three prompts of a small model in one step, odd chunk and cache lengths
        dict(name="prefill-3-ragged", op="prefill", seqs=3, lo=37, hi=1001, past_lo=5, past_hi=700, nh=8, nkv=2,
             hd=64, bs=32),
        # one 2048-token prompt from an empty cache
        dict(name="prefill-2048", op="prefill", seqs=1, lo=2048, hi=2048, past_lo=0, past_hi=0, nh=32, nkv=8, hd=128,
             bs=64),
        # the last 2048-token chunk of a prompt that fills the window
        dict(name="prefill-2048-at-6144", op="prefill", seqs=1, lo=2048, hi=2048, past_lo=6144, past_hi=6144, nh=32,
             nkv=8, hd=128, bs=64),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "append", "gather", "decode", "decode", "prefill", "prefill"])
    nh, nkv, hd = rng.choice([(32, 8, 128), (8, 2, 64), (16, 2, 256), (8, 8, 128), (24, 8, 128), (16, 1, 64)])
    bs = rng.choice([16, 32, 64])
    if op == "plan":
        seqs = _log(rng, 1, 512)
        decode = rng.randint(max(0, seqs - 64), seqs)
        lo, hi = sorted((_log(rng, 1, 30000), _log(rng, 1, 30000)))
        clo, chi = sorted((_log(rng, 1, 512), _log(rng, 1, 512)))
        return dict(op=op, seqs=seqs, decode=decode, lo=lo, hi=hi, chunk_lo=clo, chunk_hi=chi, bs=bs)
    if op == "append":
        rot = rng.choice([hd, hd // 2, 64])
        rows = _log(rng, 1, 2048 if (nh + 2 * nkv) * hd <= 6144 else 1024)
        return dict(op=op, rows=rows, nh=nh, nkv=nkv, hd=hd, rot=rot, style=rng.randint(0, 1),
                    norm=rng.random() < 0.5, bs=bs, pos=_log(rng, 1, 8192))
    if op == "gather":
        rows = _log(rng, 1, 65536 * 8 * 128 // (nkv * hd * 4))
        return dict(op=op, rows=rows, nkv=nkv, hd=hd, bs=bs, blocks=-(-rows // bs) + rng.randint(1, 100))
    if op == "decode":
        rows = _log(rng, 1, 64)
        top = min(8192 * 32 // rows, 32768) * 1024 // (nkv * hd) if rows <= 16 else 4096
        lo, hi = sorted((_log(rng, 1, min(top, 40000)), _log(rng, 1, min(top, 40000))))
        return dict(op=op, rows=rows, nh=nh, nkv=nkv, hd=hd, bs=bs, lo=lo, hi=hi)
    if hd == 256:
        nh, nkv, hd = 16, 4, 128
    seqs = rng.randint(1, 4)
    lo, hi = sorted((_log(rng, 2, 2048 // seqs), _log(rng, 2, 2048 // seqs)))
    plo, phi = sorted((_log(rng, 1, 6144 // seqs), _log(rng, 1, 6144 // seqs)))
    return dict(op=op, seqs=seqs, lo=lo, hi=hi, past_lo=plo - 1, past_hi=phi - 1, nh=nh, nkv=nkv, hd=hd, bs=bs)


def _spread(n, lo, hi):
    """``n`` lengths from ``lo`` to ``hi``, even over the logarithm (the case alone decides them)."""
    if n == 1:
        return [hi]
    return [int(round((lo + 1) * ((hi + 1) / (lo + 1)) ** (i / (n - 1)))) - 1 for i in range(n)]


def _plan_lens(c):
    """(tokens cached, new tokens) of every request: decoding requests first."""
    chunks = c["seqs"] - c["decode"]
    new = [1] * c["decode"] + (_spread(chunks, c["chunk_lo"], c["chunk_hi"]) if chunks else [])
    return _spread(c["seqs"], c["lo"], c["hi"]), new


def _prefill_lens(c):
    """(tokens cached before the chunk, chunk rows) of every sequence."""
    return _spread(c["seqs"], c["past_lo"], c["past_hi"])[::-1], _spread(c["seqs"], c["lo"], c["hi"])


# ---- inputs ------------------------------------------------------------------------------------
def _random_cache(g, blocks, nkv, bs, hd):
    """A cache as quantised activations leave it: codes peaked at the middle of their range, scales
    spread over an octave or so, centres off zero."""
    units, codes, pairs = bs // 16, 16 * hd, 32 * (hd // 64)
    cache = torch.empty(blocks, nkv, units, 18 * hd, dtype=torch.uint8, device=DEV)
    step = max(1, (1 << 27) // (nkv * units * codes))
    for b in range(0, blocks, step):
        part = cache[b:b + step]
        shape = (part.shape[0], nkv, units, codes)
        lo = (torch.randn(shape, device=DEV, generator=g).mul_(2.8).add_(7.5)).round_().clamp_(0, 15)
        hi = (torch.randn(shape, device=DEV, generator=g).mul_(2.8).add_(7.5)).round_().clamp_(0, 15)
        part[..., :codes] = (lo + 16 * hi).to(torch.uint8)
        s = torch.exp(0.4 * torch.randn(*shape[:3], pairs, device=DEV, generator=g)) * 0.3
        z = 0.2 * torch.randn(*shape[:3], pairs, device=DEV, generator=g)
        part[..., codes:] = torch.stack([s, z], -1).half().reshape(*shape[:3], 2 * pairs).view(torch.uint8)
    return cache


def _tables(g, ctx, bs):
    """Random distinct blocks for sequences of ``ctx`` tokens: (block tables, blocks in all)."""
    need = [-(-max(1, n) // bs) for n in ctx]
    width, total = max(need) + 1, sum(need) + 3
    perm = torch.randperm(total, device=DEV, generator=g).int()
    tab, at = torch.zeros(len(ctx), width, dtype=torch.int32, device=DEV), 0
    for i, n in enumerate(need):
        tab[i, :n] = perm[at:at + n]
        at += n
    return tab, total


def _queries(g, rows, nh, hd):
    """bf16 queries; heads differ in how peaked their attention is."""
    t = torch.exp(torch.linspace(math.log(0.5), math.log(4.0), nh, device=DEV))
    return (torch.randn(rows, nh, hd, device=DEV, generator=g) * t[:, None]).bfloat16()


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = np.random.RandomState(seed % (1 << 31))
    c, op = dict(case), case["op"]
    s = {"case": c}
    if op == "plan":
        cached, new = _plan_lens(c)
        cached = [cached[i] for i in r.permutation(len(cached))]
        n, bs = c["seqs"], c["bs"]
        width = -(-(max(cached) + max(new)) // bs) + 1
        have = [-(-a // bs) for a in cached]
        perm = torch.randperm(sum(have) + n + sum(new), device=DEV, generator=g).int()
        tab, at = torch.zeros(n + 4, width, dtype=torch.int32, device=DEV), 0
        rows = r.permutation(n + 4)[:n]
        for i in range(n):
            tab[int(rows[i]), :have[i]] = perm[at:at + have[i]]
            at += have[i]
        total = sum(new)
        need = sum(-(-(a + b) // bs) - -(-a // bs) for a, b in zip(cached, new))
        cap = -(-(total + 7) // 8) * 8
        out = torch.zeros(4, cap, dtype=torch.int32, device=DEV)
        s.update(seq_rows=_ints(rows), cached=_ints(cached), new=_ints(new), tables=tab, free=perm[at:].contiguous(),
                 out=out, taken=torch.zeros(1, dtype=torch.int32, device=DEV), total=total, need=need,
                 status=torch.zeros(1, dtype=torch.int32, device=DEV), host=(rows, cached, new))
    elif op == "append":
        R, nh, nkv, hd, bs, rot = (c[k] for k in ("rows", "nh", "nkv", "hd", "bs", "rot"))
        qkv = torch.randn(R, (nh + 2 * nkv) * hd, device=DEV, generator=g)
        # a few key channels are several times larger than the rest, as rotated keys have them
        boost = torch.ones(nh + 2 * nkv, hd, device=DEV)
        boost[nh:nh + nkv, ::29] = 4.0
        qkv *= boost.reshape(-1)
        blocks = -(-R // bs) + 5
        tok = torch.randperm(blocks, device=DEV, generator=g)[: -(-R // bs)]
        slots = (tok[:, None] * bs + torch.arange(bs, device=DEV)[None]).reshape(-1)[:R].int()
        i = torch.arange(rot // 2, dtype=torch.float64, device=DEV)
        ang = torch.arange(c["pos"] + 1, dtype=torch.float64, device=DEV)[:, None] * (10000.0 ** (-2.0 * i / rot))
        s.update(qkv=qkv, slots=slots, rope=torch.stack([torch.cos(ang), torch.sin(ang)], -1).float(),
                 positions=torch.randint(0, c["pos"] + 1, (R,), device=DEV, generator=g).int(),
                 q_norm=(1 + 0.1 * torch.randn(hd, device=DEV, generator=g)) if c["norm"] else None,
                 k_norm=(1 + 0.1 * torch.randn(hd, device=DEV, generator=g)) if c["norm"] else None,
                 cache=torch.zeros(blocks, nkv, bs // 16, 18 * hd, dtype=torch.uint8, device=DEV),
                 q=torch.empty(R, nh, hd, dtype=torch.bfloat16, device=DEV),
                 k=torch.empty(R, nkv, hd, dtype=torch.bfloat16, device=DEV),
                 v=torch.empty(R, nkv, hd, dtype=torch.bfloat16, device=DEV))
    elif op == "gather":
        R, nkv, hd, bs = (c[k] for k in ("rows", "nkv", "hd", "bs"))
        tok = torch.randperm(c["blocks"], device=DEV, generator=g)[: -(-R // bs)]
        s.update(cache=_random_cache(g, c["blocks"], nkv, bs, hd),
                 slots=(tok[:, None] * bs + torch.arange(bs, device=DEV)[None]).reshape(-1)[:R].int(),
                 k=torch.empty(R, nkv, hd, dtype=torch.bfloat16, device=DEV),
                 v=torch.empty(R, nkv, hd, dtype=torch.bfloat16, device=DEV))
    else:
        nh, nkv, hd, bs = (c[k] for k in ("nh", "nkv", "hd", "bs"))
        if op == "decode":
            ctx = [_spread(c["rows"], c["lo"], c["hi"])[i] for i in r.permutation(c["rows"])]
            row_seq, row_ctx, spans = list(range(len(ctx))), ctx, [(i, 1) for i in range(len(ctx))]
        else:
            past, new = _prefill_lens(c)
            ctx = [a + b for a, b in zip(past, new)]
            row_seq = [i for i, n in enumerate(new) for _ in range(n)]
            row_ctx = [past[i] + j + 1 for i, n in enumerate(new) for j in range(n)]
            spans = [(i, n) for i, n in enumerate(new)]
        tab, blocks = _tables(g, ctx, bs)
        R = len(row_seq)
        s.update(cache=_random_cache(g, blocks, nkv, bs, hd), tables=tab, row_seq=_ints(row_seq),
                 row_ctx=_ints(row_ctx), q=_queries(g, R, nh, hd), top=max(ctx), spans=spans,
                 out=torch.empty(R, nh * hd, dtype=torch.bfloat16, device=DEV),
                 # a row's place in a [sequences, longest chunk] grid (the plain form's padding)
                 place=torch.tensor([i * max(n for _, n in spans) + j for i, n in spans for j in range(n)],
                                    device=DEV))
    return s


# ---- the plain form: elementary operations in 32 bits -------------------------------------------
def _unpack(u, hd):
    """fp32 keys and values [..., 16, hd] of cache units [..., 18 * hd]."""
    lead, kc = u.shape[:-1], 8 * hd
    planes, words = max(1, hd // 128), min(4, hd // 32)

    def nibbles(b):  # [..., 2 (e), 2 (p high), 2 (p low)] of 4-byte words
        w = b.reshape(*b.shape[:-1], -1, 4)
        return torch.stack([w & 15, w >> 4], -1).reshape(*w.shape[:-1], 2, 2, 2)

    n = len(lead)
    k = nibbles(u[..., :kc]).reshape(*lead, planes, 16, 4, words, 2, 2, 2)
    # dims in order plane, i, t, p high, p low, e
    k = k.permute(*range(n), n + 1, n, n + 3, n + 2, n + 5, n + 6, n + 4).reshape(*lead, 16, hd)
    v = nibbles(u[..., kc:2 * kc]).reshape(*lead, hd // 64, 8, 4, 2, 2, 2, 2, 2)
    # tokens in order h, t, e; dims in order plane, i, g, p high, p low
    v = v.permute(*range(n), n + 4, n + 2, n + 5, n, n + 3, n + 1, n + 6, n + 7).reshape(*lead, 16, hd)
    sc = u[..., 2 * kc:].contiguous().view(torch.float16).float().reshape(*lead, 2, 16, hd // 64, 2)

    def value(code, p):
        code = code.reshape(*lead, 16, hd // 64, 64).float()
        return (p[..., 1:] + p[..., :1] * (code - 8.0)).reshape(*lead, 16, hd)

    return value(k, sc[..., 0, :, :, :]), value(v, sc[..., 1, :, :, :])


def _plain_plan(s):
    c = s["case"]
    bs, dev = c["bs"], s["new"].device
    cached, new, free, tab = s["cached"].long(), s["new"].long(), s["free"], s["tables"]
    seq = s["seq_rows"].long()
    b0, b1 = (cached + bs - 1) // bs, (cached + new + bs - 1) // bs
    ids = torch.arange(c["seqs"], device=dev)
    j = torch.arange(s["need"], device=dev)
    owner = torch.repeat_interleave(ids, b1 - b0, output_size=s["need"])
    base = torch.cumsum(b1 - b0, 0) - (b1 - b0)
    tab[seq[owner], b0[owner] + j - base[owner]] = free[: s["need"]]
    row = torch.arange(s["total"], device=dev)
    owner = torch.repeat_interleave(ids, new, output_size=s["total"])
    pos = cached[owner] + row - (torch.cumsum(new, 0) - new)[owner]
    out, n = s["out"], s["total"]
    out[0, :n], out[1, :n], out[2, :n] = pos, seq[owner], pos + 1
    out[3, :n] = tab[seq[owner], pos // bs] * bs + pos % bs
    out[0:3, n:] = 0
    out[3, n:] = -1
    s["taken"][0] = (b1 - b0).sum()
    return {"rows": out, "tables": tab, "taken": s["taken"]}


def _rotate(x, rope, style):
    half = rope.shape[1]
    cs, sn = rope[:, None, :, 0], rope[:, None, :, 1]
    y = x.clone()
    a, b = (x[..., 0:2 * half:2], x[..., 1:2 * half:2]) if style == 0 else (x[..., :half], x[..., half:2 * half])
    ra, rb = a * cs - b * sn, a * sn + b * cs
    if style == 0:
        y[..., 0:2 * half:2], y[..., 1:2 * half:2] = ra, rb
    else:
        y[..., :half], y[..., half:2 * half] = ra, rb
    return y


def _plain_append(s):
    c = s["case"]
    R, nh, nkv, hd = (c[k] for k in ("rows", "nh", "nkv", "hd"))
    x = s["qkv"].reshape(R, nh + 2 * nkv, hd)
    q, k, v = x[:, :nh], x[:, nh:nh + nkv], x[:, nh + nkv:]
    if c["norm"]:
        q = q * torch.rsqrt((q * q).mean(-1, keepdim=True) + 1e-6) * s["q_norm"]
        k = k * torch.rsqrt((k * k).mean(-1, keepdim=True) + 1e-6) * s["k_norm"]
    rope = s["rope"][s["positions"].long()]
    q, k = _rotate(q, rope, c["style"]), _rotate(k, rope, c["style"])

    def held(x):  # the values that the 4-bit codes stand for
        x = x.reshape(R, nkv, hd // 64, 64)
        lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
        sc = ((hi - lo) / 15.0).half().float()
        z = (lo + 8.0 * sc).half().float()
        code = torch.where(sc > 0, torch.round((x - z) / sc) + 8.0, torch.full_like(x, 8.0)).clamp(0.0, 15.0)
        return (z + sc * (code - 8.0)).reshape(R, nkv, hd).bfloat16()

    return {"q": q.bfloat16(), "k": held(k), "v": held(v)}


def _plain_gather(s):
    c, slots = s["case"], s["slots"].long()
    u = s["cache"][slots // c["bs"], :, slots % c["bs"] // 16]
    k, v = _unpack(u, c["hd"])
    at = (slots % 16).reshape(-1, 1, 1, 1).expand(-1, c["nkv"], 1, c["hd"])
    return {"k": k.gather(2, at)[:, :, 0].bfloat16(), "v": v.gather(2, at)[:, :, 0].bfloat16()}


def _plain_attention(s):
    c = s["case"]
    nh, nkv, hd, bs, top = c["nh"], c["nkv"], c["hd"], c["bs"], s["top"]
    n, G = -(-top // bs), c["nh"] // c["nkv"]
    S, m = len(s["spans"]), max(k for _, k in s["spans"])
    u = s["cache"][s["tables"][:, :n].long()]               # [S, blocks, nkv, units, bytes]
    k, v = _unpack(u.transpose(1, 2), hd)                   # [S, nkv, blocks, units, 16, hd]
    k, v = (t.reshape(S, nkv, -1, hd)[:, :, :top] for t in (k, v))
    q = torch.zeros(S * m, nh, hd, device=DEV)
    q[s["place"]] = s["q"].float()
    ctx = torch.zeros(S * m, dtype=torch.int64, device=DEV)
    ctx[s["place"]] = s["row_ctx"].long()
    q = q.reshape(S, m, nkv, G, hd).permute(0, 2, 1, 3, 4).reshape(S, nkv, m * G, hd)
    p = torch.matmul(q, k.transpose(-1, -2)).reshape(S, nkv, m, G, top) * (1.0 / math.sqrt(hd))
    seen = torch.arange(top, device=DEV) < ctx.reshape(S, 1, m, 1, 1)
    p = torch.where(seen, p, torch.full((), -math.inf, device=DEV))
    p = torch.exp(p - p.amax(-1, keepdim=True).clamp_min(-3e38))
    p = (p / p.sum(-1, keepdim=True).clamp_min(1e-38)).reshape(S, nkv, m * G, top)
    o = torch.matmul(p, v).reshape(S, nkv, m, G, hd).permute(0, 2, 1, 3, 4).reshape(S * m, nh * hd)
    return o[s["place"]].bfloat16()


def run(state):
    s, c = state, state["case"]
    op = c["op"]
    if not own:
        if op == "plan":
            return _plain_plan(s)
        if op == "append":
            return _plain_append(s)
        if op == "gather":
            return _plain_gather(s)
        return _plain_attention(s)
    kv4, ws = _kv4()
    if op == "plan":
        o = s["out"]
        kv4.plan_rows(s["seq_rows"], s["cached"], s["new"], s["tables"], c["bs"], o[0], o[1], o[2], o[3],
                      free_blocks=s["free"], taken=s["taken"], status=s["status"])
        return {"rows": o, "tables": s["tables"], "taken": s["taken"]}
    if op == "append":
        kv4.rope_append(s["qkv"], s["positions"], s["slots"], s["rope"], c["rot"], c["style"], s["q"], s["cache"],
                        c["nh"], c["nkv"], c["hd"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=1e-6)
        kv4.gather(s["cache"], s["slots"], s["k"], s["v"])
        return {"q": s["q"], "k": s["k"], "v": s["v"]}
    if op == "gather":
        kv4.gather(s["cache"], s["slots"], s["k"], s["v"])
        return {"k": s["k"], "v": s["v"]}
    attend = kv4.attention_decode if op == "decode" else kv4.attention_prefill
    attend(s["q"], s["cache"], s["tables"], s["row_seq"], s["row_ctx"], 1.0 / math.sqrt(c["hd"]), ws,
           out_bf16=s["out"])
    return s["out"]


def work(case):
    c, op = case, case["op"]
    if op == "plan":
        cached, new = _plan_lens(c)
        need = sum(-(-(a + b) // c["bs"]) - -(-a // c["bs"]) for a, b in zip(cached, new))
        rows = sum(new)
        # lengths in, four values a row out, the slots' table entries in, new blocks in and out
        return {"bytes": 12 * c["seqs"] + 16 * rows + 4 * -(-rows // c["bs"]) + 8 * need, "flops": 8 * rows}
    if op == "append":
        rows, kv = c["rows"], c["rows"] * c["nkv"] * c["hd"]
        read = rows * ((c["nh"] + 2 * c["nkv"]) * c["hd"] * 4 + c["rot"] * 4 + 8)
        held = kv * 9 // 8                      # K and V at 4.5 bits
        return {"bytes": read + rows * c["nh"] * c["hd"] * 2 + 2 * held + 4 * kv,
                "flops": rows * (c["nh"] + c["nkv"]) * c["hd"] * 3 + 16 * kv}
    if op == "gather":
        kv = c["rows"] * c["nkv"] * c["hd"]
        return {"bytes": kv * 9 // 8 + 4 * kv + 4 * c["rows"], "flops": 4 * kv}
    if op == "decode":
        tokens = pairs = sum(_spread(c["rows"], c["lo"], c["hi"]))
        rows = c["rows"]
    else:
        past, new = _prefill_lens(c)
        tokens, rows = sum(past) + sum(new), sum(new)
        pairs = sum(n * a + n * (n + 1) // 2 for a, n in zip(past, new))
    return {"bytes": tokens * c["nkv"] * c["hd"] * 9 // 8 + rows * c["nh"] * c["hd"] * 4,
            "flops": 4 * pairs * c["nh"] * c["hd"]}


# ---- the definition in 64 bits ------------------------------------------------------------------
def _held64(unit_bytes, token, hd):
    """Keys and values of tokens ``token`` (int64 [N], place in the unit) from units [N, heads, bytes],
    read code by code: every (token, head dim) is looked up at its byte and nibble."""
    d = torch.arange(hd, device=DEV)[None]
    t = token[:, None]

    def code(byte, odd):
        b = torch.gather(unit_bytes, 2, byte[:, None, :].expand(-1, unit_bytes.shape[1], -1)).long()
        return torch.where(odd[:, None, :].bool(), b // 16, b % 16).double()

    row = min(hd, 128) // 2  # bytes of one token's keys in a plane
    r = d % 128
    nib = (r % 8) // 2 + 4 * (r % 2)
    kb = (d // 128) * 16 * row + t * row + ((r // 8) % 4) * (row // 4) + (r // 32) * 4 + nib // 2
    kc = code(kb, (nib % 2).expand_as(kb))
    r = d % 64
    nib = (r % 4) + 4 * (t % 2)
    vb = 8 * hd + (d // 64) * 512 + ((r % 32) // 4) * 64 + ((t % 8) // 2) * 16 + (r // 32) * 8 + (t // 8) * 4 + nib // 2
    vc = code(vb, nib % 2)
    out = []
    for which, cd in ((0, kc), (1, vc)):
        at = 16 * hd + which * hd + t * (hd // 16) + (d // 64) * 4
        raw = [torch.gather(unit_bytes, 2, (at + i)[:, None, :].expand(-1, unit_bytes.shape[1], -1)).int()
               for i in range(4)]
        s, z = ((raw[i] + 256 * raw[i + 1]).to(torch.int16).view(torch.float16).double() for i in (0, 2))
        out.append(z + s * (cd - 8))
    return out


def _tokens64(s, seq, n):
    """Keys and values [n, heads, hd] of the first ``n`` tokens of table row ``seq``."""
    c, t = s["case"], torch.arange(n, device=DEV)
    blk = s["tables"][seq].long()[t // c["bs"]]
    return _held64(s["cache"][blk, :, t % c["bs"] // 16], t % 16, c["hd"])


def exact(case, seed):
    s, c, op = prepare(case, seed), case, case["op"]
    if op == "plan":
        rows, cached, new = s["host"]
        tab, free = s["tables"].cpu().numpy().copy(), s["free"].cpu().numpy()
        out, used, at, bs = np.zeros(tuple(s["out"].shape), np.int32), 0, 0, c["bs"]
        out[3] = -1
        for q, a, n in zip(rows, cached, new):
            for p in range(a, a + n):
                if p // bs >= -(-a // bs) and (p == a or p % bs == 0):
                    tab[q, p // bs] = free[used]
                    used += 1
                out[:, at] = p, q, p + 1, tab[q, p // bs] * bs + p % bs
                at += 1
        return {"rows": out, "tables": tab, "taken": np.array([used], np.int32)}
    if op == "append":
        R, nh, nkv, hd, half = c["rows"], c["nh"], c["nkv"], c["hd"], c["rot"] // 2
        x = s["qkv"].double().reshape(R, -1, hd)
        if c["norm"]:
            for a, b, w in ((0, nh, s["q_norm"]), (nh, nh + nkv, s["k_norm"])):
                x[:, a:b] = x[:, a:b] / torch.sqrt(x[:, a:b].pow(2).sum(-1, keepdim=True) / hd + 1e-6) * w.double()
        z = s["rope"].double()[s["positions"].long()]
        z = torch.complex(z[..., 0], z[..., 1])[:, None]
        i = torch.arange(half, device=DEV)
        a, b = (2 * i, 2 * i + 1) if c["style"] == 0 else (i, i + half)
        turned = torch.complex(x[:, :nh + nkv, a], x[:, :nh + nkv, b]) * z
        x[:, :nh + nkv, a], x[:, :nh + nkv, b] = turned.real, turned.imag

        def held(y):
            out = torch.empty_like(y)
            for j in range(0, hd, 64):
                part = y[..., j:j + 64]
                lo = part.min(-1, keepdim=True).values
                sc = ((part.max(-1, keepdim=True).values - lo) / 15).to(torch.float16).double()
                mid = (lo + 8 * sc).to(torch.float16).double()
                code = torch.floor((part - mid) / sc.clamp_min(1e-30) + 0.5).clamp(-8, 7)
                out[..., j:j + 64] = mid + sc * code
            return out

        return {"q": x[:, :nh], "k": held(x[:, nh:nh + nkv]), "v": held(x[:, nh + nkv:])}
    if op == "gather":
        slots = s["slots"].long()
        k, v = torch.empty(2, c["rows"], c["nkv"], c["hd"], dtype=torch.float64, device=DEV)
        for i in range(0, c["rows"], 8192):
            t = slots[i:i + 8192]
            k[i:i + 8192], v[i:i + 8192] = _held64(s["cache"][t // c["bs"], :, t % c["bs"] // 16], t % 16, c["hd"])
        return {"k": k, "v": v}
    nh, nkv, hd = c["nh"], c["nkv"], c["hd"]
    G, at, parts = nh // nkv, 0, []
    for seq, n in s["spans"]:
        ctx = s["row_ctx"][at:at + n].long()
        k, v = _tokens64(s, seq, int(ctx.max()))
        q = s["q"][at:at + n].double()
        o = torch.zeros(n, nh, hd, dtype=torch.float64, device=DEV)
        late = torch.arange(k.shape[0], device=DEV)[None] >= ctx[:, None]
        for h in range(nh):
            w = torch.softmax((q[:, h] @ k[:, h // G].T / math.sqrt(hd)).masked_fill(late, -math.inf), -1)
            o[:, h] = w @ v[:, h // G]
        parts.append(o.reshape(n, nh * hd))
        at += n
    return torch.cat(parts)
