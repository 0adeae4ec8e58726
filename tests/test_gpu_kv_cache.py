"""GPU tests of the paged cache beside its operators: its bookkeeping does not wait for
the GPU, and scoring leaves no pools behind."""

import pytest
import torch

from evo2_flash_b200.kv_cache import PagedKVCache

pytestmark = pytest.mark.gpu


def test_bookkeeping_does_not_wait_for_the_gpu():
    """Under torch's check for synchronising calls: a prompt, forks, and decode steps
    that copy a shared page, take new ones and grow the pools."""
    c = PagedKVCache(2, heads=2, head_dim=64, page_size=16)
    prompt, steps = 40, 600
    positions = [torch.arange(prompt, device="cuda")]
    positions += [torch.full((3,), prompt + i, device="cuda") for i in range(steps)]
    torch.cuda.synchronize()
    mode = torch.cuda.get_sync_debug_mode()
    torch.cuda.set_sync_debug_mode("error")
    try:
        made = [c.step([(0, prompt, 0, 0)], positions[0])]
        c.fork(0, 1, prompt)
        c.fork(0, 2, prompt)
        made += [c.step([(r, r + 1, r, prompt + i) for r in range(3)], positions[1 + i]) for i in range(steps)]
    finally:
        torch.cuda.set_sync_debug_mode(mode)
    # what the copies brought, each from pinned memory of its own until it is done
    assert made[0].seq_lens.tolist() == [prompt] and made[0].starts.tolist() == [0, prompt]
    for i, step in enumerate(made[1:]):
        assert step.seq_lens.tolist() == [prompt + i + 1] * 3 and step.starts is None
    last = made[-1]
    assert last.table.tolist() == [c._pages[r] for r in range(3)]
    assert last.shared["shared_lens"].tolist() == [32] and last.shared["group_start"].tolist() == [0, 3]
    assert c.layer(1)[1].shape == (128, 16, 2, 64)


@pytest.fixture(scope="module")
def native():
    from evo2_flash_b200.model import StripedHyena2, StripedHyena2Config

    m = StripedHyena2(StripedHyena2Config.small(hidden=256, use_fp8_input_projections=False, native_blocks=True),
                      device="cuda")
    m.load_tensors(m.random_tensors(23))
    return m


def _seqs(*lens):
    g = torch.Generator().manual_seed(1)
    return [torch.randint(65, 70, (n,), generator=g) for n in lens]


@pytest.mark.parametrize("budget", [None, 50])
def test_scoring_leaves_no_pools(native, budget):
    seqs = _seqs(120, 30, 70)
    for run in (native.score, native.token_logprobs,
                lambda s, b: list(native.prefill_steps(s, b)),
                lambda s, b: list(native.prefill_steps(s, b, {1}))):
        run(seqs, budget)
        assert native.cache._pages == {}
        assert all(t is None for pool in native.cache._pools for t in pool)
    list(native.prefill_steps(seqs, budget, keep_cache=True))
    assert sorted(native.cache._pages) == [0, 1, 2]  # kept for decode steps
    native.release_all()


@pytest.mark.parametrize("limit,sharing,called", [(2048, True, True), (9, True, True), (8, False, True),
                                                  (5, False, True), (4, False, False)])
def test_sequences_and_groups_beyond_one_call(native, monkeypatch, limit, sharing, called):
    """Five sequences, two of which share a prompt: with the three others' groups nine in
    all.  Where the groups are too many, the sequences read for themselves."""
    from evo2_flash_b200 import ops
    from tests.helpers import REL_TOL, max_rel_err

    seqs, seen, paged = _seqs(100, 20, 30, 40), [], ops.paged_attention

    def spy(*args, **kw):
        seen.append("shared_lens" in kw)
        return paged(*args, **kw)

    def step(n):
        monkeypatch.setattr(ops, "PAGED_ATTENTION_REQUESTS", n)
        with torch.no_grad():
            list(native.prefill_steps(seqs, keep_cache=True, state_blocks=6))
            native.fork(0, 4, 100)
            monkeypatch.setattr(ops, "paged_attention", spy)
            try:
                seen.clear()
                return native.decode_step([65] * 5, [100, 100, 20, 30, 40], [0, 4, 1, 2, 3])
            finally:
                monkeypatch.setattr(ops, "paged_attention", paged)
                native.release_all()

    want, got = step(2048), step(limit)
    layers = len(native.cfg.attn_layer_idxs)
    assert len(seen) == (layers if called else 0) and all(x == sharing for x in seen)
    assert max_rel_err(got.float().cpu(), want.float().cpu()) < 2 * REL_TOL
