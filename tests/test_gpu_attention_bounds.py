"""GPU tests of ops.paged_attention for lengths beyond the page table and token
ranges beyond the rows of q: queries stay at their positions, what does not exist
is left out, and the error flags tell (1: pages, 2: token ranges)."""

import pytest
import torch

from tests.test_gpu_attention import BF, DEV, Batch, attend, sharing, widen

pytestmark = pytest.mark.gpu


def check_rows(b, out, r, rows, first):
    """Rows `rows` of request r, whose first query sees the keys before `first`."""
    k, v = b.keys[r]
    ref, tol = attend(b.q[rows], k, v, first, b.dim ** -0.5)
    assert ((out[rows].double() - ref).abs() <= tol).all(), r


@pytest.mark.parametrize("heads,kv_heads", [(2, 2), (8, 2), (5, 1)])
@pytest.mark.parametrize("over", [1, 6, 2 ** 31 - 65])
def test_lengths_beyond_the_table(heads, kv_heads, over):
    """Four queries over a table of 64 positions, a length of 64 + over: all but those
    of `over` see all 64 keys."""
    b = Batch([(4, 64), (2, 40), (1, 64)], heads, kv_heads, page=16)
    lens = b.seq_lens.clone()
    lens[0] += over
    out = b.call(seq_lens=lens)
    assert int(b.flags) == 1
    check_rows(b, out, 0, slice(0, 4), 64 - 3 + min(over, 1000))
    check_rows(b, out, 1, slice(4, 6), 39)
    check_rows(b, out, 2, slice(6, 7), 64)


@pytest.mark.parametrize("over", [1, 3])
def test_lengths_beyond_a_wide_table(over):
    """The same where the plan has a kernel of its own."""
    keys = 65536
    b = widen(Batch([(4, 300), (1, 70), (3, 9), (1, 16), (2, 33)], 4, 4, page=16), keys)
    page = int(b.table[0, 0])
    b.table[0, 19:] = page  # every further page holds the first one's keys
    k, v = b.keys[0]
    at = torch.arange(keys, device=DEV)
    at = torch.where(at < 304, at, at % 16)
    b.k[int(b.table[0, 18]), 12:], b.v[int(b.table[0, 18]), 12:] = k[:4], v[:4]
    at[300:304] = torch.arange(4, device=DEV)
    b.keys[0] = (k[at], v[at])
    lens = b.seq_lens.clone()
    lens[0] = keys + over
    out = b.call(seq_lens=lens)
    assert int(b.flags) == 1
    check_rows(b, out, 0, slice(0, 4), keys - 3 + over)
    check_rows(b, out, 2, slice(5, 8), 7)


@pytest.mark.parametrize("members", [6, 40, 150])
def test_lengths_beyond_the_table_in_a_group(members):
    """Each kind of kernel for the shared run."""
    b = Batch([(2, 1024)] * members, 4, 4, page=16, groups=[(range(members), 640)])
    lens = b.seq_lens.clone()
    lens[1] += 1
    lens[4] += 700
    out = b.call(seq_lens=lens, **sharing((members, 640)))
    assert int(b.flags) == 1
    for r, over in ((0, 0), (1, 1), (4, 700), (5, 0)):
        check_rows(b, out, r, slice(2 * r, 2 * r + 2), 1023 + over)


def test_a_length_at_the_end_of_the_table_is_no_error():
    b = Batch([(4, 64), (1, 64)], 2, 2, page=16)
    b.check(b.call())


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("grouped", [False, True])
def test_token_ranges_beyond_the_rows(wide, grouped):
    """Request 4 claims six tokens where q has four more rows: those four sit at the
    first four of its six positions."""
    groups = [([3, 4], 32)] if grouped else []
    b = Batch([(1, 5), (2, 40), (1, 17), (1, 90), (6, 200), (0, 0)], 4, 2, page=16, groups=groups)
    if wide:
        widen(b, 2 ** 18)
    starts = b.starts.clone()
    b.q = b.q[:9].contiguous()
    kw = dict(shared_lens=torch.tensor([32], device=DEV), group_start=torch.tensor([3, 5], device=DEV)) if grouped else {}
    out = b.call(query_start_loc=starts, **kw)
    assert int(b.flags) == 2
    check_rows(b, out, 4, slice(5, 9), 195)
    check_rows(b, out, 1, slice(1, 3), 39)
    check_rows(b, out, 3, slice(4, 5), 90)


def test_decreasing_token_ranges_are_flagged():
    b = Batch([(1, 5), (2, 40), (1, 17)], 4, 2, page=16)
    b.call(query_start_loc=torch.tensor([0, 3, 2, 4], dtype=torch.int32, device=DEV))
    assert int(b.flags) == 2
