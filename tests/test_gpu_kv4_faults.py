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
