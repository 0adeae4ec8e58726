"""StripedHyena2 with native_blocks (paged cache, kv_append, paged_attention,
gated_mlp) against the same model on torch's attention and MLP, and generate's
shared prompts.

The two differ in roundings only (an MLP rounded once instead of three times, a
rotation in one fp32 pass): blocks are held to the path's bar, scores to the
NLL bars of the other model tests, 1e-3 for the mean over the sequences and 2e-3
for one.  (A token's log-probability moves by a few 1e-3 with the roundings of its
hidden state, 2^-8 of each element, independently from token to token: 5e-3 / 8 for
the mean of the shortest sequence's 63, three times that within 2e-3.)"""

import pytest
import torch

from tests.helpers import REL_TOL, max_rel_err
from tests.test_api_cpu import _dna, _incremental_vs_prefill

pytestmark = pytest.mark.gpu
NLL_TOL = 1e-3


@pytest.fixture(scope="module")
def models():
    from evo2_flash_b200.model import StripedHyena2, StripedHyena2Config

    plain = StripedHyena2(StripedHyena2Config.small(hidden=256, use_fp8_input_projections=False), device="cuda")
    native = StripedHyena2(StripedHyena2Config.small(hidden=256, use_fp8_input_projections=False,
                                                     native_blocks=True), device="cuda")
    t = plain.random_tensors(23)
    plain.load_tensors(t)
    native.load_tensors(t)
    return plain, native


def _tokens(n, seed):
    return torch.tensor(list(_dna(n, seed).encode()), dtype=torch.long)


@pytest.mark.parametrize("budget", [None, 300, 50])
def test_scores_match_torch_blocks(models, budget):
    plain, native = models
    seqs = [_tokens(n, 60 + n) for n in (700, 1, 130, 64, 333)]
    a = plain.token_logprobs(seqs, max_tokens_per_step=budget)
    b = native.token_logprobs(seqs, max_tokens_per_step=budget)
    assert native.cache._pages == {}
    assert all(x.shape == y.shape and torch.isfinite(y).all() for x, y in zip(a, b))
    c, d = plain.score(seqs, max_tokens_per_step=budget), native.score(seqs, max_tokens_per_step=budget)
    for first, second in ((c, d), ([-float(x.mean()) for x in a], [-float(x.mean()) for x in b])):
        gaps = [x - y for x, y in zip(first, second) if x == x]
        assert len(gaps) == 4 and first[1] != first[1] and second[1] != second[1]  # one token: nothing to score
        assert abs(sum(gaps) / 4) <= NLL_TOL, gaps
        assert max(map(abs, gaps)) <= 2 * NLL_TOL, gaps


def test_decode_steps_match_one_pass(models):
    _, native = models
    p, toks = _tokens(200, 21).tolist(), _tokens(16, 22).tolist()
    errs = _incremental_vs_prefill(native, p, toks)
    assert max(errs) < REL_TOL, errs


def test_blocks_match_torch_blocks_on_the_same_input(models):
    """Attention (a packed step, a continued chunk, single tokens) and MLP layer by
    layer; further on, the random-init stack's cubic gates amplify the roundings."""
    plain, native = models
    pa, na = plain.layers[3].mixer, native.layers[3].mixer
    g = torch.Generator(device="cuda").manual_seed(4)
    with torch.no_grad():
        for segs in ([(0, 100, 0, 0), (100, 130, 1, 0)], [(0, 70, 0, 100), (70, 75, 1, 30)],
                     [(0, 1, 1, 35), (1, 2, 0, 170)], [(0, 4, 0, 171), (4, 5, 1, 36)]):
            T = segs[-1][1]
            x = torch.randn(T, 256, generator=g, device="cuda").to(torch.bfloat16)
            pos = torch.cat([torch.arange(p0, p0 + b - a) for a, b, _, p0 in segs]).cuda()
            want = pa(x, pos, segs)
            got = na(x, pos, native.cache.step(segs, pos))
            assert max_rel_err(got.float().cpu(), want.float().cpu()) < REL_TOL
        for i in (0, 1):
            got, want = native.layers[i].mlp(x), plain.layers[i].mlp(x)
            assert max_rel_err(got.float().cpu(), want.float().cpu()) < REL_TOL
    plain.release_all()
    native.release_all()


def test_mlp_hooks_still_see_the_projections(models):
    from evo2_flash_b200.api import Evo2

    plain, native = models
    ids = _tokens(64, 50)[None]
    names = ["blocks.1.mlp.l1", "blocks.1.mlp.l3", "blocks.3.inner_mha_cls"]
    a, ea = Evo2(plain)(ids, return_embeddings=True, layer_names=names)
    b, eb = Evo2(native)(ids, return_embeddings=True, layer_names=names)
    for n in names:
        assert ea[n].shape == eb[n].shape
        assert max_rel_err(eb[n].float().cpu(), ea[n].float().cpu()) < 2 * REL_TOL


def test_fork_continues_like_the_original(models):
    _, native = models
    p = _tokens(150, 8)
    with torch.no_grad():
        list(native.prefill_steps([p], keep_cache=True, state_blocks=4))
        native.fork(0, 1, 150)
        native.fork(0, 2, 150)
        for step in range(30):  # over the end of a page
            t = [65, 65, 71]
            h = native.decode_step(t, [150 + step] * 3, [0, 1, 2])
            assert torch.equal(h[0], h[1])
            assert step < 2 or not torch.equal(h[0], h[2])
    native.release_all()


def test_more_sequences_than_one_call_takes(models, monkeypatch):
    from evo2_flash_b200 import ops

    _, native = models
    with torch.no_grad():
        outs = []
        for limit in (2048, 4):
            monkeypatch.setattr(ops, "PAGED_ATTENTION_REQUESTS", limit)
            list(native.prefill_steps([_tokens(20 + i, i) for i in range(5)], keep_cache=True))
            outs.append(native.decode_step([65] * 5, [20 + i for i in range(5)], range(5)))
    native.release_all()
    assert max_rel_err(outs[1].float().cpu(), outs[0].float().cpu()) < 2 * REL_TOL


def test_hooks_before_a_projection_run(models):
    _, native = models
    mlp, seen = native.layers[1].mlp, []
    x = torch.randn(3, 256, device="cuda").to(torch.bfloat16)
    hook = mlp.l2.register_forward_pre_hook(lambda m, args: seen.append(args[0].shape))
    try:
        mlp(x)
    finally:
        hook.remove()
    assert seen == [x.shape]


@pytest.mark.parametrize("temperature", [0.0, 1.0])
def test_generate_samples_of_one_prompt(models, temperature):
    """Four samples of one prompt among others: the results of the prompts given one
    by one, every sequence where its prompt stands."""
    from evo2_flash_b200.api import Evo2

    _, native = models
    evo = Evo2(native)
    x, y = _dna(90, 70), _dna(40, 71)
    prompts = [x, y, x, x, y, x]
    out = evo.generate(prompts, n_tokens=12, temperature=temperature, top_k=4, seed=5, verbose=0)
    assert [len(v) for v in out.token_ids] == [12] * 6
    for i, (p, toks, mean) in enumerate(zip(prompts, out.token_ids, out.logprobs_mean)):
        full = torch.tensor(evo.tokenizer.tokenize(p) + toks)
        lp = native.token_logprobs([full])[0][len(p) - 1:]
        # 12 tokens a prompt, log-probabilities a few 1e-3 apart in steps of other lengths
        assert abs(float(lp.mean()) - mean) <= 4 * NLL_TOL, i
    if temperature == 0.0:
        assert out.token_ids[0] == out.token_ids[2] == out.token_ids[3] == out.token_ids[5]
        assert out.token_ids[1] == out.token_ids[4]
    assert native.cache._pages == {}
