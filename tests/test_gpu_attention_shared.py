"""GPU tests of ops.paged_attention's kernels for shared runs of many rows, where a
row's running maximum moves along the run: growing keys, scores of any size and
sign, NaN keys, pages out of range.  Formulas, batches and tolerances are those of
test_gpu_attention.py: 2^-8 (|o| + A) + 2 (2 e + 2^-19) A, from the roundings alone."""

import pytest
import torch

from tests.test_gpu_attention import BF, DEV, Batch, attend, sharing

pytestmark = pytest.mark.gpu

# (heads, kv heads, dim, page, samples, shared keys): one and two row tiles of 128
# query rows a key/value head, several key tiles an item (32 key/value heads leave a
# run of 24 tiles five pieces or fewer), boxes of a page and of a whole key tile
ONE_TILE = [(32, 32, 128, 64, 24, 3000), (32, 32, 64, 16, 40, 2560), (64, 32, 128, 128, 12, 2700)]
TWO_TILES = [(64, 32, 128, 64, 70, 2600), (32, 32, 64, 48, 150, 2400)]
SHAPES = ONE_TILE + TWO_TILES


def samples_of_one_prompt(heads, kv_heads, dim, page, samples, shared, seed=0):
    reqs = [(1, shared + 1 + 3 * (i % 5)) for i in range(samples)]
    return Batch(reqs, heads, kv_heads, dim, page, groups=[(range(samples), shared)], seed=seed)


def rewrite(b, change):
    """keys[r] = change(keys, positions) of every request, in its pages too."""
    for r, (k, v) in enumerate(b.keys):
        k = change(k, torch.arange(len(k), device=DEV)).to(BF)
        b.keys[r] = (k, v)
        for j in range(-(-len(k) // b.page)):
            rows = k[j * b.page:(j + 1) * b.page]
            b.k[int(b.table[r, j]), :len(rows)] = rows


def check_some(b, out, scale=None, keep=None):
    """Every seventh request (for the oracle's time), over its keys `keep` alone."""
    scale = b.dim ** -0.5 if scale is None else scale
    for r in range(0, len(b.requests), 7):
        k, v = b.keys[r]
        rows = torch.arange(len(k), device=DEV) if keep is None else keep(len(k))
        ref, tol = attend(b.q[r:r + 1], k[rows], v[rows], len(rows), scale)
        assert torch.isfinite(ref).all() and torch.isfinite(tol).all()
        bad = (out[r:r + 1].double() - ref).abs() - tol
        assert (bad <= 0).all(), (r, float(bad.max()))
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("steps", [3, 12])
def test_keys_that_grow_along_the_run(shape, steps):
    """Scores rise by some 20 a step for half of the rows, so that their maximum
    moves at several tiles of an item, and fall for the other half, warp by warp
    mixed."""
    b = samples_of_one_prompt(*shape)
    shared, u = shape[5], torch.ones(b.dim, device=DEV)
    up = torch.arange(b.tokens, device=DEV) % 2 * 2 - 1
    # q.k / sqrt(D) changes by 20 for each step: c g sqrt(D) = 20
    b.q.add_((2.0 * up[:, None, None] * u).to(BF))
    rewrite(b, lambda k, at: k + (10.0 / b.dim ** 0.5 * (at * steps // shared))[:, None, None] * u)
    check_some(b, b.call(**sharing((shape[4], shared))))


@pytest.mark.parametrize("shape", SHAPES)
def test_large_scores(shape):
    b = samples_of_one_prompt(*shape, seed=1)
    b.q[::2] *= 40
    check_some(b, b.call(**sharing((shape[4], shape[5]))))


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("scale", [0.0, -1.5])
def test_zero_and_negative_scales(shape, scale):
    b = samples_of_one_prompt(*shape, seed=2)
    check_some(b, b.call(scale=scale, **sharing((shape[4], shape[5]))), scale)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("at", [0, 1000, 2300])
def test_a_nan_key_reaches_its_head_alone(shape, at):
    b = samples_of_one_prompt(*shape, seed=3)
    kw = sharing((shape[4], shape[5]))
    clean = b.call(**kw)
    b.k[int(b.table[0, at // b.page]), at % b.page, 3] = float("nan")
    out = b.call(**kw)
    per = shape[0] // shape[1]
    hit = torch.zeros(shape[0], dtype=torch.bool, device=DEV)
    hit[3 * per:4 * per] = True
    assert torch.isnan(out[:, hit]).all()
    assert torch.equal(out[:, ~hit], clean[:, ~hit])


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("first,n", [(0, 1), (0, 10), (7, 3), (-1, 1)])
def test_bad_pages_of_the_run_are_flagged_and_not_read(shape, first, n):
    """Pages out of range at the start of the run (a whole key tile and more), in its
    middle and at its end: their keys are left out, the rest as ever."""
    b = samples_of_one_prompt(*shape, seed=4)
    shared, pages = shape[5], shape[5] // b.page
    first = first if first >= 0 else pages + first
    b.table[:, first:first + n:2] = b.k.shape[0]
    b.table[:, first + 1:first + n:2] = -5
    out = b.call(**sharing((shape[4], shared)))
    assert int(b.flags) == 1
    lo, hi = first * b.page, (first + n) * b.page

    def keep(length):
        at = torch.arange(length, device=DEV)
        return at[(at < lo) | (at >= hi)]

    check_some(b, out, keep=keep)


def far_below_zero(b):
    """Scores of -300 (natural) and less in the shared run, so that their weights
    against a maximum of 0 would vanish; values around 1."""
    u = torch.ones(b.dim, device=DEV)
    b.q.mul_(0.5).add_((3.0 * u).to(BF))
    rewrite(b, lambda k, at: 0.5 * k - 100.0 / b.dim ** 0.5 * u)
    for r, (k, v) in enumerate(b.keys):
        v = (v + 1).to(BF)
        b.keys[r] = (k, v)
        for j in range(-(-len(v) // b.page)):
            rows = v[j * b.page:(j + 1) * b.page]
            b.v[int(b.table[r, j]), :len(rows)] = rows


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("keys", [128, 400])
def test_low_scores_behind_bad_pages(shape, keys):
    """A run whose first key tile has no key at all: the others count all the same."""
    b = samples_of_one_prompt(*shape, seed=5)
    far_below_zero(b)
    n = -(-keys // b.page)
    b.table[:, :n] = -1
    out = b.call(**sharing((shape[4], shape[5])))
    assert int(b.flags) == 1
    check_some(b, out, keep=lambda length: torch.arange(n * b.page, length, device=DEV))


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("keys", [100, 128, 400])
def test_low_scores_behind_scores_of_minus_infinity(shape, keys):
    """The first keys score -inf (weight 0), for some rows a whole tile of them; the
    next ones -300.  (The reference leaves the keys of no weight out.)"""
    b = samples_of_one_prompt(*shape, seed=6)
    far_below_zero(b)

    def minus_inf(k, at):
        k = k.clone()
        k[:keys, :, 0] = float("-inf")
        return k

    rewrite(b, minus_inf)
    b.q[:, :, 0] = b.q[:, :, 0].abs() + 0.1
    out = b.call(**sharing((shape[4], shape[5])))
    assert int(b.flags) == 0
    check_some(b, out, keep=lambda length: torch.arange(keys, length, device=DEV))
