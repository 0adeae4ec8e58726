"""The paged key/value cache's host bookkeeping, on the CPU: page tables, growth,
forks with copy on write, and the shared runs it reports."""

import pytest
import torch

from evo2_flash_b200.kv_cache import PagedKVCache


def cache(page=16, layers=2):
    return PagedKVCache(layers, heads=2, head_dim=4, page_size=page, device="cpu", dtype=torch.float32)


def write(c, table, row, positions, value):
    for i in range(c.layers):
        k, v = c.layer(i)
        for p in positions:
            k[table[row, p // c.page_size], p % c.page_size] = value + p + 1000 * i
            v[table[row, p // c.page_size], p % c.page_size] = -(value + p)


def read(c, table, row, n, layer=0):
    k, _ = c.layer(layer)
    return torch.stack([k[table[row, p // c.page_size], p % c.page_size] for p in range(n)])[:, 0, 0]


def test_pages_follow_the_lengths_and_come_back():
    c = cache()
    c.extend(0, 0, 40)
    c.extend(1, 0, 16)
    table, shared = c.table([0, 1])
    assert table.shape == (2, 3) and table.dtype == torch.int32 and shared == {}
    used = table[0].tolist() + table[1, :1].tolist()
    assert len(set(used)) == 4
    c.extend(1, 16, 17)
    assert c.table([1])[0].shape == (1, 2)
    c.release(0)
    c.extend(2, 0, 33)  # freed pages are used again
    assert set(c.table([2])[0][0].tolist()) <= set(range(16))
    with pytest.raises(ValueError, match="cannot continue"):
        c.extend(2, 60, 61)
    with pytest.raises(ValueError, match="multiple of 16"):
        cache(page=24)


def test_growth_keeps_what_is_stored():
    c = cache()
    c.extend(0, 0, 30)
    write(c, c.table([0])[0], 0, range(30), 5.0)
    before = read(c, c.table([0])[0], 0, 30)
    c.extend(1, 0, 16 * 100)
    assert c.layer(0)[0].shape[0] >= 102
    assert torch.equal(read(c, c.table([0])[0], 0, 30), before)
    assert torch.equal(read(c, c.table([0])[0], 0, 30, layer=1), before + 1000)


def test_beginning_anew_releases_the_old_pages():
    c = cache()
    for _ in range(50):
        c.extend(0, 0, 160)
    assert c.layer(0)[0].shape[0] <= 32


def test_fork_shares_until_written():
    c = cache()
    n = 40  # two whole pages and half of one
    c.extend(0, 0, n)
    write(c, c.table([0])[0], 0, range(n), 0.0)
    c.fork(0, 1, n)
    c.fork(0, 2, n)
    table, shared = c.table([0, 1, 2])
    assert torch.equal(table[0], table[1]) and torch.equal(table[0], table[2])
    assert shared["shared_lens"].tolist() == [48] and shared["group_start"].tolist() == [0, 3]
    c.extend(1, n, n + 1)  # writes into the third page: its own copy
    table, shared = c.table([0, 1, 2])
    assert torch.equal(table[0, :2], table[1, :2]) and table[0, 2] != table[1, 2]
    assert torch.equal(table[0], table[2])
    assert shared["shared_lens"].tolist() == [32]
    write(c, table, 1, [n], 500.0)
    assert torch.equal(read(c, table, 1, n), read(c, table, 0, n))
    c.extend(0, n, n + 1)
    c.extend(2, n, n + 1)
    assert len(set(c.table([0, 1, 2])[0][:, 2].tolist())) == 3
    c.release(0)  # the others keep the shared pages
    assert torch.equal(read(c, c.table([2])[0], 0, n), torch.arange(n, dtype=torch.float32))
    with pytest.raises(ValueError, match="fewer"):
        c.fork(1, 3, 1000)


def test_shared_runs_of_several_groups():
    c = cache()
    for s, n in ((0, 64), (10, 20), (20, 33)):
        c.extend(s, 0, n)
    for d in (1, 2):
        c.fork(0, d, 64)
    c.fork(20, 21, 33)
    order = [0, 1, 2, 10, 20, 21]
    _, shared = c.table(order)
    assert shared["group_start"].tolist() == [0, 3, 4, 6]
    assert shared["shared_lens"].tolist() == [64, 0, 48]
    assert c.table([10, 0])[1] == {}
    assert c.table([1, 10, 2])[1] == {}  # not side by side: nothing read together


def test_step_arguments():
    c = cache()
    step = c.step([(0, 3, 5, 0), (3, 5, 7, 0)], torch.arange(5))
    assert list(step) == [(0, 3, 5, 0), (3, 5, 7, 0)]
    assert step.starts.tolist() == [0, 3, 5] and step.seq_lens.tolist() == [3, 2]
    assert step.longest == 3 and step.positions.dtype == torch.int32
    step = c.step([(0, 1, 5, 3), (1, 2, 7, 2)], torch.tensor([3, 2]))
    assert step.starts is None and step.seq_lens.tolist() == [4, 3] and step.longest == 1


def test_native_blocks_need_cuda_and_a_head_size():
    from evo2_flash_b200.model import StripedHyena2, StripedHyena2Config
    from tests.helpers import OracleMixer

    with pytest.raises(ValueError, match="CUDA"):
        StripedHyena2(StripedHyena2Config.small(hidden=128, native_blocks=True), device="cpu",
                      mixer_factory=OracleMixer)


def test_growth_holds_one_old_tensor_too_many_at_most(monkeypatch):
    """A pool's old tensor is dropped before the next pool's new one is made."""
    import weakref

    c = cache(layers=3)
    c.extend(0, 0, 16)
    old = [weakref.ref(t) for pool in c._pools for t in pool]
    held, empty = [], torch.empty

    def spy(*args, **kw):
        held.append(sum(r() is not None for r in old))
        return empty(*args, **kw)

    monkeypatch.setattr(torch, "empty", spy)
    c.extend(1, 0, 16 * 40)
    assert held[:6] == [6, 5, 4, 3, 2, 1]
    assert all(r() is None for r in old)


def test_growth_that_fails_leaves_the_cache_as_it_was(monkeypatch):
    c = cache(layers=2)
    c.extend(0, 0, 30)
    write(c, c.table([0])[0], 0, range(30), 5.0)
    before, made, empty = read(c, c.table([0])[0], 0, 30), [], torch.empty

    def fails(*args, **kw):
        made.append(1)
        if len(made) == 2:
            raise torch.OutOfMemoryError("no room")
        return empty(*args, **kw)

    monkeypatch.setattr(torch, "empty", fails)
    with pytest.raises(torch.OutOfMemoryError):
        c.extend(1, 0, 16 * 100)
    monkeypatch.setattr(torch, "empty", empty)
    k, v = c.layer(0)
    assert k.shape == v.shape
    assert torch.equal(read(c, c.table([0])[0], 0, 30), before)
    c.release(1)
    c.extend(2, 0, 16 * 100)
    assert torch.equal(read(c, c.table([0])[0], 0, 30, layer=1), before + 1000)
    assert c.layer(0)[0].shape == c.layer(1)[1].shape


def test_positions_that_were_never_written_are_not_skipped():
    """Inside a sequence's last page too: what lies between would be read by attention."""
    c = cache(page=64)
    c.extend(0, 0, 10)
    with pytest.raises(ValueError, match="has 10 positions, cannot continue at 11"):
        c.extend(0, 11, 12)
    with pytest.raises(ValueError, match="has 0 positions, cannot continue at 5"):
        c.extend(1, 5, 6)
    assert 1 not in c._pages
    for length in (11, 64, -1):
        with pytest.raises(ValueError, match="fewer than"):
            c.fork(0, 1, length)
    c.fork(0, 1, 10)
    c.fork(0, 2, 7)
    c.extend(1, 10, 11)
    with pytest.raises(ValueError, match="has 7 positions"):
        c.extend(2, 10, 11)
    c.extend(0, 10, 14)
    c.extend(0, 12, 13)  # back, as after rejected tokens; what was written may be continued
    c.extend(0, 14, 15)
    c.extend(0, 0, 3)  # anew
    with pytest.raises(ValueError, match="has 3 positions"):
        c.extend(0, 4, 5)
    c.release(0)
    with pytest.raises(ValueError, match="has 0 positions"):
        c.extend(0, 3, 4)
