"""Paged KV cache in 4 bits: Python surface of kv4_cache.cu, kv4_decode.cu and kv4_prefill.cu.

A layer's cache is uint8 ``[blocks, kv_heads, block_size / 16, 18 * head_dim]`` (``cache_shape``):
16 tokens of one head per unit, a 4-bit code per value and one float16 pair (s, c) per token and 64
head dims; a value is ``c + s * (code - 8)``, 4.5 bits in all against 16 of the bf16 cache.

A step runs ``plan_rows`` (positions, sequences, contexts and slots of its rows, and the new blocks
of its block tables, from the request lengths), then per layer ``rope_append`` and
``attention_decode`` (rows that are one token of a sequence each) or ``attention_prefill`` (runs of
rows of one sequence). ``gather`` reads tokens back as bf16 rows.

Every function launches on the current CUDA stream. Kernels never follow bad device-side indices.
``plan_rows`` and the attention report them in a status word (the ``status`` argument,
``Workspace.status``: 4); ``rope_append`` skips such rows and ``gather`` gives zeros, without a word. A
context past the end of its table row is taken as the table row's length.

Parity: crates/hawking-core/shaders/mha.metal (int4 KV decode, per-row scales),
workspace/docs/reference/env_flags.md:29-35 (the int4 KV mode).
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from .._ext import kernels
from . import PDL, launches

HEAD_DIMS = (64, 128, 256)
PREFILL_HEAD_DIMS = (64, 128)
MAX_GROUP = 16  # query heads per kv head


def unit_bytes(head_dim: int) -> int:
    """Bytes of 16 tokens of one kv head (keys and values)."""
    if head_dim not in HEAD_DIMS:
        raise ValueError(f"4-bit KV cache: head_dim must be one of {HEAD_DIMS}, not {head_dim}")
    return 18 * head_dim


def cache_shape(num_blocks: int, n_kv_heads: int, block_size: int, head_dim: int) -> Tuple[int, int, int, int]:
    """Shape of one layer's cache tensor (uint8)."""
    if block_size <= 0 or block_size % 16:
        raise ValueError(f"4-bit KV cache: block_size must be a multiple of 16, not {block_size}")
    return num_blocks, n_kv_heads, block_size // 16, unit_bytes(head_dim)


def unit_tokens(head_dim: int) -> torch.Tensor:
    """The token (0 to 15) that each byte of a unit belongs to: no byte holds parts of two."""
    unit_bytes(head_dim)
    t, groups = torch.arange(16), head_dim // 64
    keys = t.repeat_interleave(min(head_dim, 128) // 2).repeat(max(1, head_dim // 128))
    # value words [group][g 8][t 4][i 2][h 2] hold tokens 8 h + 2 t (low half) and 8 h + 2 t + 1 (high half)
    values = t.view(2, 4, 2).permute(1, 0, 2)[None, None, :, None, :, :, None].expand(groups, 8, 4, 2, 2, 2, 2)
    pairs = t.repeat_interleave(4 * groups).repeat(2)
    return torch.cat([keys, values.reshape(-1), pairs])


class Workspace:
    """What the attention launches of one stream share: the device status word, the partial results of
    rows that several CTAs work on, and their arrival counters (zero between launches). Use one
    workspace per stream: launches that share one must be ordered.

    ``wait_polls`` bounds the kernels' waits: one that runs out sets the status word to 3, leaves the
    launch's outputs undefined and needs a ``reset`` before the next launch."""

    def __init__(self, device="cuda"):
        self.device = torch.device(device)
        self.sms = torch.cuda.get_device_properties(self.device).multi_processor_count
        floats, counters = kernels().kv4_workspace_sizes(self.sms)
        self.status = torch.zeros(1, dtype=torch.int32, device=device)
        self.part = torch.empty(floats, dtype=torch.float32, device=device)
        self.counters = torch.zeros(counters, dtype=torch.int32, device=device)
        self.wait_polls = kernels().KV4_WAIT_POLLS

    def reset(self):
        """Clear the status word and the counters (after a launch reported a failed wait)."""
        self.status.zero_()
        self.counters.zero_()


def plan_rows(seq_rows: torch.Tensor, cached: torch.Tensor, new: torch.Tensor, block_tables: torch.Tensor,
              block_size: int, positions: torch.Tensor, row_seq: torch.Tensor, row_ctx: torch.Tensor,
              slots: torch.Tensor, free_blocks: Optional[torch.Tensor] = None,
              taken: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None):
    """Rows of a step from the request lengths, on the GPU.

    Request i (block-table row ``seq_rows[i]``, ``cached[i]`` tokens in the cache, ``new[i]`` to
    append; int32, at most 8192 requests) owns the next ``new[i]`` rows. Row outputs (int32, one
    length): ``positions``, ``row_seq`` (block-table row), ``row_ctx`` (position + 1) and ``slots``
    (block * block_size + offset); rows past the last get 0, 0, 0 and -1, which ``rope_append`` and
    the attention kernels skip. With ``free_blocks`` the blocks that the new tokens need are taken
    from it in order, request by request, and written into ``block_tables``; ``taken`` gets their
    number. Without it the tables must already hold them.

    A request that does not fit its table row (or has a negative length or a bad row) gets no rows;
    rows that do not fit the outputs are dropped, rows whose block is missing (a negative entry of the
    table or the list, or a list too short) or too large for an int32 slot get slot -1. Each sets
    ``status`` to 4 (bad argument)."""
    launches.add()
    kernels().kv4_plan(seq_rows, cached, new, block_tables, block_size, positions, row_seq, row_ctx, slots,
                       free_blocks, taken, status, PDL)


def rope_append(qkv: torch.Tensor, positions: torch.Tensor, slots: Optional[torch.Tensor], rope: torch.Tensor,
                rot_dim: int, style: int, q_out: torch.Tensor, cache: torch.Tensor, nh: int, nkv: int, hd: int,
                bias: Optional[torch.Tensor] = None, q_norm: Optional[torch.Tensor] = None,
                k_norm: Optional[torch.Tensor] = None, eps: float = 1e-6,
                block_tables: Optional[torch.Tensor] = None, row_seq: Optional[torch.Tensor] = None):
    """RoPE q / k (optional bias and per-head q / k RMSNorm), q as bf16 rows, k / v quantised into
    the cache at ``slots`` (or, when slots is None, at the slot the block table maps each row's
    position to). A row with a negative or foreign slot stores nothing, a row with a position
    outside ``rope`` is left alone.

    Groups of 64 dims: s = f16((max - min) * (1 / 15)), c = f16(min + 8 s), code =
    rint((x - c) / s) + 8 in 0..15 (8 where s is 0), each operation rounded to fp32. Finite values beyond +-65024 are clamped to it; a group with
    a NaN or an infinity reads back as NaN."""
    launches.add()
    kernels().kv4_append(qkv, positions, slots, rope, rot_dim, style, q_out, cache, nh, nkv, hd, bias, q_norm, k_norm,
                         eps, block_tables, row_seq, PDL)


def gather(cache: torch.Tensor, slots: torch.Tensor, k: Optional[torch.Tensor], v: Optional[torch.Tensor]):
    """The keys and values of token ``slots`` as bf16 ``[slots, kv_heads, head_dim]`` rows (either
    may be None); a slot outside the cache gives zeros."""
    launches.add()
    kernels().kv4_gather(cache, slots, k, v, PDL)


def attention_decode(q: torch.Tensor, cache: torch.Tensor, block_tables: torch.Tensor, row_seq: torch.Tensor,
                     row_ctx: torch.Tensor, scale: float, ws: Workspace, out: Optional[torch.Tensor] = None,
                     out_bf16: Optional[torch.Tensor] = None, sinks: Optional[torch.Tensor] = None):
    """Attention of bf16 queries ``[rows, heads, head_dim]`` over the first ``row_ctx`` cached tokens
    of each row's sequence, for rows that are one token of a sequence each (any mix is right, long
    runs of one sequence are faster in ``attention_prefill``). ``out`` (fp32) and / or ``out_bf16``:
    ``[rows, heads * head_dim]``. A row with no context gives zeros. ``sinks`` (fp32 ``[heads]``): a logit
    per head that takes weight and adds nothing (NaN makes the head NaN, +infinity zero)."""
    launches.add()
    kernels().kv4_attention(False, q, cache, block_tables, row_seq, row_ctx, scale, out, out_bf16, sinks, ws.status,
                            ws.part, ws.counters, ws.sms, PDL, ws.wait_polls)


def attention_prefill(q: torch.Tensor, cache: torch.Tensor, block_tables: torch.Tensor, row_seq: torch.Tensor,
                      row_ctx: torch.Tensor, scale: float, ws: Workspace, out: Optional[torch.Tensor] = None,
                      out_bf16: Optional[torch.Tensor] = None, sinks: Optional[torch.Tensor] = None):
    """``attention_decode`` for runs of rows of one sequence (prompt chunks), causal through
    ``row_ctx``; head_dim 64 or 128."""
    launches.add()
    kernels().kv4_attention(True, q, cache, block_tables, row_seq, row_ctx, scale, out, out_bf16, sinks, ws.status,
                            ws.part, ws.counters, ws.sms, PDL, ws.wait_polls)
