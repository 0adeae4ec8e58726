"""GPU parity of ops.kv_append and ops.paged_attention against the formulas in
fp64 (plain torch, this file), at the sizes, masks and layouts where they can go
wrong.

Tolerances.  A rounding to bf16 is off by at most 2^-8 of the value.
kv_append: one rounding of a cos - b sin; the fp32 products, sum, cos and sin add
at most 8 * 2^-24 (|a| + |b|).
paged_attention: one rounding of the result, and one of each softmax weight to
bf16 before the value product: 2^-8 (|o| + A) with A = sum_j w_j |v_j|.  A score
of D exact products summed in fp32 is off by at most e = D 2^-23 |q|.|k| scale,
a weight (over its sum, off alike) by 2e + 2^-19 of itself (exp2, the fp32 sums
and the joining factors), which adds that times 2A."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16


def rope(x, pos, theta):
    """x (T, h, D) at positions (T,): fp64."""
    half = x.shape[-1] // 2
    f = theta ** (-torch.arange(half, dtype=torch.float64, device=x.device) / half)
    ang = pos.double()[:, None] * f
    c, s = ang.cos()[:, None], ang.sin()[:, None]
    a, b = x[..., :half].double(), x[..., half:].double()
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def rope_tol(x, ref):
    half = x.shape[-1] // 2
    ab = x[..., :half].double().abs() + x[..., half:].double().abs()
    return ref.abs() * 2.0 ** -8 + 8 * 2.0 ** -24 * torch.cat([ab, ab], -1)


def attend(q, k, v, first, scale):
    """Query i of q (n, heads, D) over k, v (len, kv heads, D), seeing keys
    < first + i: (result, tolerance) in fp64."""
    n, heads, D = q.shape
    per = heads // k.shape[1]
    o = torch.zeros(n, heads, D, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(o)
    for i in range(n):
        m = min(first + i, k.shape[0])
        if m <= 0:
            continue
        kk = k[:m].double().repeat_interleave(per, 1)
        vv = v[:m].double().repeat_interleave(per, 1)
        qq = q[i].double()
        s = torch.einsum("hd,khd->hk", qq, kk) * scale
        w = torch.softmax(s, -1)
        o[i] = torch.einsum("hk,khd->hd", w, vv)
        A = torch.einsum("hk,khd->hd", w, vv.abs())
        e = D * 2.0 ** -23 * abs(scale) * torch.einsum("hd,khd->hk", qq.abs(), kk.abs()).amax(-1, keepdim=True)
        tol[i] = 2.0 ** -8 * (o[i].abs() + A) + 2 * (2 * e + 2.0 ** -19) * A
    return o, tol


class Batch:
    """Requests (new tokens, keys) in groups sharing their first `shared` keys,
    on randomly ordered pages.  Every row that no request holds is NaN."""

    def __init__(self, requests, heads, kv_heads, dim=128, page=64, groups=None, seed=0, head_major=True,
                 spare=3, tail=0, uniform=True):
        g = torch.Generator(device=DEV).manual_seed(seed)
        rnd = lambda *s: torch.randn(*s, generator=g, device=DEV).to(BF)  # noqa: E731
        self.requests, self.page, self.dim, self.heads = requests, page, dim, heads
        groups = groups or []
        member = {r: (gi, sh) for gi, (members, sh) in enumerate(groups) for r in members}
        width = max([1] + [-(-n // page) for _, n in requests])
        need = []
        for r, (_, n) in enumerate(requests):
            pages = -(-n // page)
            whole = min(member[r][1] // page, pages) if r in member else 0
            need.append((whole, pages))
        total = sum(p for _, p in need) + sum(-(-sh // page) for _, sh in groups) + spare
        ids = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).tolist()
        self.spare_page = ids.pop()
        shape = (total, kv_heads, page, dim) if head_major else (total, page, kv_heads, dim)
        nan = lambda: torch.full(shape, float("nan"), dtype=BF, device=DEV)  # noqa: E731
        self.k, self.v = nan(), nan()
        if head_major:
            self.k, self.v = self.k.transpose(1, 2), self.v.transpose(1, 2)
        shared_pages = [[ids.pop() for _ in range(sh // page)] for _, sh in groups]
        shared_rows = [(rnd(sh, kv_heads, dim), rnd(sh, kv_heads, dim)) for _, sh in groups]
        self.table = torch.full((len(requests), width), self.spare_page, dtype=torch.int32)
        self.keys = []
        for r, (_, n) in enumerate(requests):
            whole, pages = need[r]
            gi = member[r][0] if r in member else None
            row = (shared_pages[gi][:whole] if gi is not None else []) + [ids.pop() for _ in range(pages - whole)]
            self.table[r, :pages] = torch.tensor(row, dtype=torch.int32)
            kk, vv = rnd(n, kv_heads, dim), rnd(n, kv_heads, dim)
            if gi is not None:
                m = min(n, member[r][1])
                kk[:m], vv[:m] = shared_rows[gi][0][:m], shared_rows[gi][1][:m]
            self.keys.append((kk, vv))
            for j in range(pages):
                rows = slice(j * page, min(n, (j + 1) * page))
                self.k[row[j], :rows.stop - rows.start] = kk[rows]
                self.v[row[j], :rows.stop - rows.start] = vv[rows]
        self.table = self.table.to(DEV)
        starts = [0]
        for n, _ in requests:
            starts.append(starts[-1] + n)
        self.tokens = starts[-1]
        self.starts = torch.tensor(starts, dtype=torch.int32, device=DEV)
        self.q = rnd(self.tokens + tail, heads, dim)
        self.seq_lens = torch.tensor([n for _, n in requests], dtype=torch.int32, device=DEV)
        self.flags = torch.zeros(1, dtype=torch.int32, device=DEV)

    def call(self, **kw):
        from evo2_flash_b200 import ops

        if any(n != 1 for n, _ in self.requests):
            kw.setdefault("query_start_loc", self.starts)
        kw.setdefault("error_flags", self.flags)
        return ops.paged_attention(kw.pop("q", self.q), self.k, self.v, self.table,
                                   kw.pop("seq_lens", self.seq_lens), **kw)

    def check(self, out, scale=None):
        scale = self.dim ** -0.5 if scale is None else scale
        at = 0
        for (n, length), (k, v) in zip(self.requests, self.keys):
            ref, tol = attend(self.q[at:at + n], k, v, length - n + 1, scale)
            got = out[at:at + n].double()
            assert torch.isfinite(got).all(), (n, length)
            bad = (got - ref).abs() - tol
            assert (bad <= 0).all(), (n, length, float(bad.max()))
            at += n
        assert int(self.flags) == 0


def sharing(*groups):
    """shared_lens and group_start of consecutive groups (members, shared)."""
    start = [0]
    for m, _ in groups:
        start.append(start[-1] + m)
    return dict(shared_lens=torch.tensor([s for _, s in groups], dtype=torch.int32, device=DEV),
                group_start=torch.tensor(start, dtype=torch.int32, device=DEV))


# ---------------------------------------------------------------- append
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(4, 4, 128, 64), (8, 2, 64, 16), (6, 1, 128, 48)])
@pytest.mark.parametrize("in_place", [False, True])
def test_append_rotates_and_writes(heads, kv_heads, dim, page, in_place):
    from evo2_flash_b200 import ops

    b = Batch([(5, 70), (1, 1), (33, 500), (2, 2), (130, 130)], heads, kv_heads, dim, page, tail=3)
    T = b.tokens + 3
    qkv = torch.randn(T, (heads + 2 * kv_heads) * dim, device=DEV).to(BF)
    q, k, v = (x.view(T, -1, dim) for x in qkv.split([heads * dim, kv_heads * dim, kv_heads * dim], 1))
    pos = torch.cat([torch.arange(n - m, n) for m, n in b.requests] + [torch.arange(3)]).to(DEV, torch.int32)
    pos[2] = -1  # left alone
    k0, v0, q0 = b.k.clone(), b.v.clone(), qkv.clone().split([heads * dim, 2 * kv_heads * dim], 1)[0].view(T, -1, dim)
    out = q if in_place else torch.full((T, heads, dim), 7.0, dtype=BF, device=DEV)
    was = out.clone()
    assert ops.kv_append(q, k, v, pos, b.k, b.v, b.table, b.starts, rope_theta=1e4, q_out=out,
                         error_flags=b.flags) is out
    live = (pos >= 0) & (torch.arange(T, device=DEV) < b.tokens)
    ref = rope(q0, pos, 1e4)
    assert ((out.double() - ref).abs() <= rope_tol(q0, ref))[live].all()
    assert torch.equal(out[~live], was[~live])
    request = torch.bucketize(torch.arange(T, device=DEV), b.starts[1:].long(), right=True).clamp(max=4)
    kref = rope(k, pos, 1e4)
    seen_k, seen_v = k0.clone(), v0.clone()
    for t in torch.nonzero(live)[:, 0].tolist():
        p = int(pos[t])
        pg, at = int(b.table[request[t], p // page]), p % page
        assert ((b.k[pg, at].double() - kref[t]).abs() <= rope_tol(k[t:t + 1], kref[t:t + 1])[0]).all()
        assert torch.equal(b.v[pg, at], v[t])
        seen_k[pg, at], seen_v[pg, at] = b.k[pg, at], v[t]
    assert torch.equal(b.k.view(torch.int16), seen_k.view(torch.int16))  # and nothing else
    assert torch.equal(b.v.view(torch.int16), seen_v.view(torch.int16))
    assert int(b.flags) == 0


@pytest.mark.parametrize("tokens", [1, 3, 1184, 1187])
def test_append_one_token_a_request(tokens):
    from evo2_flash_b200 import ops

    b = Batch([(1, 40)] * tokens, 2, 2, page=64, spare=1)
    k, v = torch.randn(2, tokens, 2, 128, device=DEV).to(BF)
    pos = torch.full((tokens,), 39, dtype=torch.int64, device=DEV)
    q = ops.kv_append(b.q, k, v, pos, b.k, b.v, b.table)
    ref = rope(b.q, pos, 1e4)
    assert ((q.double() - ref).abs() <= rope_tol(b.q, ref)).all()
    pages = b.table[:, 0].long()
    kref = rope(k, pos, 1e4)
    assert ((b.k[pages, 39].double() - kref).abs() <= rope_tol(k, kref)).all()
    assert torch.equal(b.v[pages, 39], v)
    assert ops.kv_append(None, k, v, pos, b.k, b.v, b.table) is None
    assert ((b.k[pages, 39].double() - kref).abs() <= rope_tol(k, kref)).all()


def test_append_far_positions():
    """At a position of two million an fp32 angle would be off by 0.1."""
    from evo2_flash_b200 import ops

    page, far = 64, 2_000_003
    q, k, v = torch.randn(3, 2, 4, 128, device=DEV).to(BF)
    kc, vc = torch.zeros(2, 2, page, 4, 128, dtype=BF, device=DEV)
    table = torch.full((1, far // page + 1), 1, dtype=torch.int32, device=DEV)
    pos = torch.tensor([far - 1, far], dtype=torch.int32, device=DEV)
    starts = torch.tensor([0, 2], dtype=torch.int32, device=DEV)
    out = ops.kv_append(q, k, v, pos, kc, vc, table, starts, rope_theta=1e6)
    for x, got in ((q, out), (k, kc[1, [(far - 1) % page, far % page]])):
        ref = rope(x, pos, 1e6)
        assert ((got.double() - ref).abs() <= rope_tol(x, ref)).all()


def test_append_bad_pages_are_flagged_and_skipped():
    from evo2_flash_b200 import ops

    q, k, v = torch.randn(3, 4, 2, 128, device=DEV).to(BF)
    kc, vc = torch.zeros(2, 3, 16, 2, 128, dtype=BF, device=DEV)
    table = torch.tensor([[0], [3], [-1], [1]], dtype=torch.int32, device=DEV)
    pos = torch.tensor([2, 2, 2, 16], dtype=torch.int32, device=DEV)  # the last is beyond the table
    flags = torch.zeros(1, dtype=torch.int32, device=DEV)
    out = ops.kv_append(q, k, v, pos, kc, vc, table, error_flags=flags)
    assert int(flags) == 1
    assert torch.equal(vc[0, 2], v[0])
    vc[0, 2] = 0
    kc[0, 2] = 0
    assert not vc.any() and not kc.any()
    ref = rope(q, pos, 1e4)
    assert ((out.double() - ref).abs() <= rope_tol(q, ref)).all()


# ---------------------------------------------------------------- attention
LENS = [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 300, 777]


@pytest.mark.parametrize("heads,kv_heads,dim,page,head_major", [
    (4, 4, 128, 64, True), (2, 2, 64, 16, False), (8, 2, 128, 48, True), (16, 1, 64, 32, True),
    (24, 1, 128, 256, False)])
def test_one_token_each(heads, kv_heads, dim, page, head_major):
    b = Batch([(1, n) for n in LENS], heads, kv_heads, dim, page, head_major=head_major)
    b.check(b.call())


@pytest.mark.parametrize("heads,kv_heads", [(4, 4), (8, 2), (5, 1)])
@pytest.mark.parametrize("requests", [
    [(4, 4), (4, 5), (4, 100), (4, 1000), (4, 20), (4, 33)],
    [(1, 1), (8, 9), (3, 400), (2, 2), (7, 64), (5, 129)],
    [(70, 70), (33, 200), (1, 5)],
    [(4, 2), (3, 1), (8, 0), (2, 500)],  # queries before the first key see nothing
])
def test_several_tokens_are_causal(heads, kv_heads, requests):
    b = Batch(requests, heads, kv_heads, page=16)
    b.check(b.call())


@pytest.mark.parametrize("shared", [0, 1, 16, 100, 128, 640, 2029])
@pytest.mark.parametrize("heads,kv_heads,new", [(4, 4, 1), (8, 2, 3), (8, 1, 1)])
def test_shared_prompt(shared, heads, kv_heads, new):
    reqs = [(new, shared + own) for own in (new, new + 1, 40, 513, 64, 100, 17, 80, 31, 33, 70)]
    b = Batch(reqs, heads, kv_heads, page=32, groups=[(range(11), shared)])
    b.check(b.call(shared_lens=torch.tensor([shared], dtype=torch.int32, device=DEV)))


@pytest.mark.parametrize("heads,kv_heads,dim", [(2, 2, 128), (16, 2, 64), (40, 1, 128)])
def test_groups_of_different_prompts(heads, kv_heads, dim):
    groups = [(3, 200), (1, 500), (5, 0), (20, 1111), (2, 48)]
    reqs, spec, r = [], [], 0
    for m, sh in groups:
        reqs += [(1 + (r + i) % 3, sh + 3 + 37 * i) for i in range(m)]
        spec.append((range(r, r + m), sh))
        r += m
    b = Batch(reqs, heads, kv_heads, dim, 16, groups=spec)
    b.check(b.call(**sharing(*groups)))


def test_many_samples_of_one_prompt():
    """More rows than one tile of any kernel, and more keys than one chunk."""
    reqs = [(1, 3000 + 1 + 7 * i) for i in range(150)]
    b = Batch(reqs, 4, 2, page=64, groups=[(range(150), 3000)])
    b.check(b.call(**sharing((150, 3000))))


@pytest.mark.parametrize("heads,kv_heads,dim", [(32, 32, 128), (32, 32, 64), (64, 8, 128)])
@pytest.mark.parametrize("samples,shared", [(18, 4100), (64, 3000), (150, 2050), (40, 1024), (64, 1024),
                                            (128, 1024), (128, 520), (300, 1024)])
def test_long_shared_runs(heads, kv_heads, dim, samples, shared):
    """Chunks of several key tiles, few and many rows, many heads."""
    reqs = [(1, shared + 1 + 3 * (i % 5)) for i in range(samples)]
    b = Batch(reqs, heads, kv_heads, dim, page=64, groups=[(range(samples), shared)])
    b.check(b.call(**sharing((samples, shared))))


def widen(b, keys):
    """Page tables that could hold `keys` keys a request."""
    more = keys // b.page - b.table.shape[1]
    pad = torch.full((len(b.requests), more), b.spare_page, dtype=torch.int32, device=DEV)
    b.table = torch.cat([b.table, pad], 1)
    return b


MIXES = [
    [(1, n) for n in LENS],
    [(1, 1), (8, 9), (3, 400), (2, 2), (7, 64), (5, 129), (1, 0), (2, 1)],
    [(70, 70), (33, 200), (1, 5), (1, 3000), (40, 41)],
    [(1, 1 + 97 * i % 700) for i in range(70)],
]


@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 4, 128), (8, 2, 64), (5, 1, 128)])
@pytest.mark.parametrize("requests", MIXES)
def test_wide_page_tables(heads, kv_heads, dim, requests):
    """Room for long contexts (half a GB a step and more), whatever the lengths are."""
    b = widen(Batch(requests, heads, kv_heads, dim, page=16), 2 ** 19)
    b.check(b.call())


@pytest.mark.parametrize("heads,kv_heads", [(4, 4), (8, 4)])
def test_wide_page_tables_and_groups(heads, kv_heads):
    groups = [(3, 200), (1, 500), (5, 0), (2, 1111), (2, 48)]
    reqs, spec, r = [], [], 0
    for m, sh in groups:
        reqs += [(1, sh + 3 + 37 * i) for i in range(m)]
        spec.append((range(r, r + m), sh))
        r += m
    b = widen(Batch(reqs, heads, kv_heads, page=16, groups=spec), 2 ** 19)
    b.check(b.call(**sharing(*groups)))


@pytest.mark.parametrize("keys", [None, 2 ** 15])
def test_many_requests(keys):
    reqs = [(1 + (i % 7 == 0), (i * 31) % 40 + 2 * (i % 3)) for i in range(2040)]
    b = Batch(reqs, 2, 2, 64, page=16)
    if keys:
        widen(b, keys)
    out = b.call()
    at = 0
    for i, (n, length) in enumerate(reqs):  # every seventh, for the oracle's time
        if i % 7 == 0:
            k, v = b.keys[i]
            ref, tol = attend(b.q[at:at + n], k, v, length - n + 1, 64 ** -0.5)
            assert ((out[at:at + n].double() - ref).abs() <= tol).all(), i
        at += n
    assert torch.isfinite(out).all() and int(b.flags) == 0


@pytest.mark.parametrize("groups,members", [(70, 3), (40, 20), (6, 150)])
def test_many_groups(groups, members):
    """More groups than the kernel of long shared runs plans for, several of its
    items a block, and pairs of its row tiles."""
    spec = [(range(members * g, members * (g + 1)), 16 * (g % 9) + 128) for g in range(groups)]
    reqs = [(1, sh + 1 + (7 * i) % 23) for m, sh in spec for i, _ in enumerate(m)]
    b = Batch(reqs, 16, 16 if groups == 6 else 1, page=16, groups=spec)
    out = b.call(**sharing(*[(len(m), sh) for m, sh in spec]))
    for i in range(0, len(reqs), 5):
        ref, tol = attend(b.q[i:i + 1], *b.keys[i], reqs[i][1], 128 ** -0.5)
        assert ((out[i:i + 1].double() - ref).abs() <= tol).all(), i
    assert int(b.flags) == 0


@pytest.mark.parametrize("samples,keys", [(6, 0), (6, 2 ** 19), (40, 0), (150, 0)])
def test_unchained_launches_and_graphs(samples, keys):
    """The same bits with and without programmatic launches, eager and replayed
    while the lengths grow, each kind of plan."""
    from evo2_flash_b200 import ops

    b = Batch([(1, 700 + 13 * i) for i in range(samples)], 4, 4, page=16, groups=[(range(samples), 688)])
    if keys:
        widen(b, keys)
    kw = sharing((samples, 688)) if samples > 6 else {}
    lens, out = b.seq_lens.clone(), torch.empty_like(b.q)
    b.call(seq_lens=lens, out=out, **kw)
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        b.call(seq_lens=lens, out=out, **kw)
    for n in (1, 60, 689, 720, 10 ** 6):
        lens.copy_(b.seq_lens.clamp(max=n))
        g.replay()
        ops.set_launch_chaining(False)
        try:
            plain = b.call(seq_lens=lens, **kw)
        finally:
            ops.set_launch_chaining(True)
        assert torch.equal(plain, out) and torch.equal(b.call(seq_lens=lens, **kw), out)
    b.check(out)


def test_other_device():
    """Tensors of another device than the current one."""
    if torch.cuda.device_count() < 2:
        pytest.skip("one device")
    b = Batch([(1, n) for n in LENS], 4, 4, page=16)
    here = b.call()
    b.k, b.v, b.table, b.flags = (t.to("cuda:1") for t in (b.k, b.v, b.table, b.flags))
    there = b.call(q=b.q.to("cuda:1"), seq_lens=b.seq_lens.to("cuda:1"))
    assert there.device.index == 1 and torch.equal(there.to(DEV), here)


def test_sharing_is_only_a_hint():
    """A shared run longer than a member's keys is cut to what all see; requests
    outside every group have their own keys only; a padded first member (no keys,
    a table of unused pages) does not count."""
    groups = [([1, 2, 3], 300)]
    b = Batch([(1, 0), (1, 310), (2, 290), (1, 700), (1, 50), (1, 0)], 4, 4, page=16, groups=groups)
    b.check(b.call(shared_lens=torch.tensor([300], dtype=torch.int32, device=DEV),
                   group_start=torch.tensor([0, 4], dtype=torch.int32, device=DEV)))
    one = b.call(shared_lens=torch.tensor([0], dtype=torch.int32, device=DEV),
                 group_start=torch.tensor([0, 4], dtype=torch.int32, device=DEV))
    b.check(one)


def test_long_context_is_split():
    b = Batch([(1, 40000), (1, 3), (2, 9000)], 2, 1, page=128)
    b.check(b.call())


@pytest.mark.parametrize("tail", [1, 37])
def test_rows_behind_the_last_request_are_left(tail):
    b = Batch([(2, 70), (1, 200), (3, 3)], 4, 2, page=16, tail=tail)
    out = torch.full((b.tokens + tail, 4, 128), 5.0, dtype=BF, device=DEV)
    assert b.call(out=out) is out
    b.check(out)
    assert (out[b.tokens:] == 5.0).all()


def test_padded_requests_give_zeros():
    b = Batch([(1, 70), (1, 0), (1, 9), (1, 0)], 4, 4, page=16, groups=[([0], 64)])
    for kw in ({}, sharing((4, 64)), sharing((1, 64))):
        out = b.call(**kw)
        b.check(out)
        assert not out[1].any() and not out[3].any()


def test_masked_values_do_not_matter():
    """A key that only later tokens of the step see may hold anything."""
    b = Batch([(4, 70), (8, 8), (2, 33)], 4, 2, page=16)
    clean = b.call()
    b.check(clean)
    for bad in (float("nan"), float("inf"), torch.finfo(BF).min):
        for r, at in ((0, 69), (1, 7), (2, 32)):
            pg = int(b.table[r, at // 16])
            b.k[pg, at % 16] = bad
            b.v[pg, at % 16] = bad
        out = b.call()
        last = b.starts[1:].long() - 1
        others = torch.ones(b.tokens, dtype=torch.bool, device=DEV)
        others[last] = False
        assert torch.equal(out[others], clean[others])


def test_scores_of_any_size():
    """Large and equal scores, infinite keys, NaN keys: what softmax gives."""
    b = Batch([(1, 100), (1, 40), (1, 33), (1, 20)], 2, 2, page=16)
    b.q[0] *= 300
    b.check(b.call())
    b.check(b.call(scale=0.0), scale=0.0)
    b.check(b.call(scale=-1.5), scale=-1.5)
    pg = int(b.table[3, 0])
    b.k[pg, 3] = float("nan")
    out = b.call()
    assert torch.isnan(out[3]).all() and torch.isfinite(out[:3]).all()


def test_strided_queries_and_output():
    b = Batch([(1, 90), (1, 17), (1, 260)], 4, 2, page=16)
    wide = torch.zeros(3, 8 * 128, dtype=BF, device=DEV)
    q = wide[:, 128:5 * 128].view(3, 4, 128)
    q.copy_(b.q)
    room = torch.zeros(4, 3, 128, dtype=BF, device=DEV)
    out = b.call(q=q, out=room.transpose(0, 1))
    b.check(out)
    b.table = torch.cat([b.table, b.table], 1)[:, :b.table.shape[1]]  # a row stride of its own
    b.check(b.call())


def test_bad_pages_are_flagged_and_not_read():
    b = Batch([(1, 100), (1, 100)], 2, 2, page=16)
    want = b.call()
    b.table[0, 2] = b.k.shape[0]
    b.table[0, 3] = -7
    out = b.call()
    assert int(b.flags) == 1
    assert torch.equal(out[1], want[1])
    k, v = b.keys[0]
    keep = torch.cat([torch.arange(32), torch.arange(64, 100)]).to(DEV)
    ref, tol = attend(b.q[:1], k[keep], v[keep], 68, 128 ** -0.5)
    assert ((out[:1].double() - ref).abs() <= tol).all()


@pytest.mark.parametrize("members,shared", [(0, 0), (3, 64), (12, 640), (40, 640), (150, 640)])
def test_in_place(members, shared):
    """out is q: rows of one piece and of several, every kind of shared run."""
    reqs = [(1 + (i % 5 == 0), shared + 2 + 61 * i % 400) for i in range(members)] + [(2, 30), (1, 3000), (1, 0)]
    groups = [(range(members), shared)] if members else []
    b = Batch(reqs, 8, 4, page=16, groups=groups)
    kw = sharing((members, shared)) if members else {}
    out = b.call(**kw)
    b.check(out)
    q = b.q.clone()
    assert b.call(q=q, out=q, **kw) is q and torch.equal(q, out)


def test_same_bits_every_time():
    reqs = [(1, 2000 + 11 * i) for i in range(40)]
    b = Batch(reqs, 4, 4, page=16, groups=[(range(40), 1999)])
    kw = sharing((40, 1999))
    out = b.call(**kw)
    for _ in range(3):
        assert torch.equal(b.call(**kw), out)


def test_graphs_serve_growing_contexts():
    """Two captured graphs, replayed in turn while the lengths grow, next to
    eager calls on another stream."""
    from evo2_flash_b200 import ops

    b = Batch([(1, 900 + 13 * i) for i in range(12)], 4, 4, page=16, groups=[(range(12), 896)])
    kw = sharing((12, 896))
    full = b.seq_lens.clone()
    lens = torch.full_like(full, 1)
    side = torch.cuda.Stream()
    outs, graphs = [], []
    for _ in range(2):
        out = torch.empty_like(b.q)
        with torch.cuda.stream(side):
            b.call(seq_lens=lens, out=out, **kw)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            b.call(seq_lens=lens, out=out, **kw)
        graphs.append(g)
        outs.append(out)
    for n in (1, 50, 897, 900):
        lens.copy_(full.clamp(max=n))
        side.wait_stream(torch.cuda.current_stream())
        for g in graphs:
            g.replay()
        with torch.cuda.stream(side):
            eager = ops.paged_attention(b.q, b.k, b.v, b.table, lens, **kw)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], eager)
    lens.copy_(full)
    graphs[1].replay()
    b.check(outs[1])


def test_offsets_beyond_32_bits():
    """Pages whose rows lie behind 2^31 elements of the cache."""
    from evo2_flash_b200 import ops

    page, heads, pages = 64, 32, 8300  # 262144 elements a page
    kc = torch.empty(pages, heads, page, 128, dtype=BF, device=DEV).transpose(1, 2)
    vc = torch.empty(pages, heads, page, 128, dtype=BF, device=DEV).transpose(1, 2)
    table = torch.tensor([[pages - 1, 0, pages - 2]], dtype=torch.int32, device=DEV)
    n = 150
    q, k, v = torch.randn(3, n, heads, 128, device=DEV).to(BF)
    pos = torch.arange(n, dtype=torch.int32, device=DEV)
    starts = torch.tensor([0, n], dtype=torch.int32, device=DEV)
    qr = ops.kv_append(q, k, v, pos, kc, vc, table, starts)
    kr = rope(k, pos, 1e4)
    for p in range(3):
        rows = slice(p * page, min(n, (p + 1) * page))
        got = kc[int(table[0, p]), :rows.stop - rows.start].double()
        assert ((got - kr[rows]).abs() <= rope_tol(k[rows], kr[rows])).all()
    kept = torch.cat([kc[int(p)] for p in table[0]])[:n]
    out = ops.paged_attention(qr[-1:].contiguous(), kc, vc, table, torch.tensor([n], device=DEV))
    ref, tol = attend(qr[-1:], kept, v, n, 128 ** -0.5)
    assert ((out.double() - ref).abs() <= tol).all()


def test_decode_run_append_then_attend():
    """A prompt and then single tokens, as a model calls the two, against fp64
    attention over the rotated keys."""
    from evo2_flash_b200 import ops

    heads, page, prompt, steps = 4, 16, 61, 6
    kc, vc = torch.zeros(2, 8, page, heads, 128, dtype=BF, device=DEV)
    table = torch.randperm(8, device=DEV).to(torch.int32)[None, :5].contiguous()
    qs, ks, vs = torch.randn(3, prompt + steps, heads, 128, device=DEV).to(BF)
    krot = rope(ks, torch.arange(prompt + steps, device=DEV), 1e4)
    at = 0
    for n in [prompt] + [1] * steps:
        rows = slice(at, at + n)
        pos = torch.arange(at, at + n, dtype=torch.int32, device=DEV)
        starts = torch.tensor([0, n], dtype=torch.int32, device=DEV)
        q = ops.kv_append(qs[rows], ks[rows], vs[rows], pos, kc, vc, table, starts)
        out = ops.paged_attention(q, kc, vc, table, torch.tensor([at + n], device=DEV), starts)
        kept = torch.cat([kc[int(p)] for p in table[0]])[:at + n]
        assert ((kept.double() - krot[:at + n]).abs() <= rope_tol(ks[:at + n], krot[:at + n])).all()
        ref, tol = attend(q, kept, vs[:at + n], at + 1, 128 ** -0.5)
        assert ((out.double() - ref).abs() <= tol).all()
        at += n


# ---------------------------------------------------------------- refusals
def test_refusals():
    from evo2_flash_b200 import ops

    b = Batch([(1, 20), (1, 30)], 4, 2, page=16)
    k, v = torch.randn(2, 2, 2, 128, device=DEV).to(BF)
    pos = torch.zeros(2, dtype=torch.int32, device=DEV)

    def refused(fn, match):
        with pytest.raises(ValueError, match=match):
            fn()

    app = lambda q=b.q, k=k, v=v, p=pos, kc=b.k, vc=b.v, t=b.table, s=None, **kw: ops.kv_append(  # noqa: E731
        q, k, v, p, kc, vc, t, s, **kw)
    refused(lambda: app(q=b.q.float()), "bf16")
    refused(lambda: app(q=b.q.cpu()), "CUDA")
    refused(lambda: app(k=k[:1]), "tokens")
    refused(lambda: app(k=k[..., :64]), "heads of 128")
    refused(lambda: app(p=pos[:1]), "positions")
    refused(lambda: app(p=pos.float()), "integers")
    refused(lambda: app(vc=b.v[:2]), "differ")
    refused(lambda: app(kc=b.k[:, :8], vc=b.v[:, :8]), "multiple of 16")
    refused(lambda: app(rope_theta=0.0), "rope_theta")
    refused(lambda: app(rope_theta=float("nan")), "rope_theta")
    refused(lambda: app(q=None, q_out=b.q), "without q")
    refused(lambda: app(s=torch.tensor([0, 1, 2, 2], device=DEV)), "page_table")
    refused(lambda: app(k=k.clone().requires_grad_()), "no backward")
    att = lambda q=b.q, kc=b.k, vc=b.v, t=b.table, n=b.seq_lens, s=None, **kw: ops.paged_attention(  # noqa: E731
        q, kc, vc, t, n, s, **kw)
    refused(lambda: att(q=b.q[:, :3]), "multiple of kv_heads")
    refused(lambda: att(q=b.q[..., :64]), "heads of 128|must have")
    refused(lambda: att(kc=b.k.half(), vc=b.v.half()), "bf16")
    refused(lambda: att(kc=b.k[..., :32], vc=b.v[..., :32], q=b.q[..., :32]), "head_dim")
    refused(lambda: att(t=b.table[:1]), "page_table")
    refused(lambda: att(s=b.starts[:2]), "query_start_loc")
    refused(lambda: att(shared_lens=pos), "group_start")
    refused(lambda: att(group_start=pos), "without shared_lens")
    refused(lambda: att(out=b.q[:1].clone()), "tokens")
    refused(lambda: att(error_flags=pos.float()), "error_flags")
    n = 2100
    refused(lambda: att(q=b.q[:1].expand(n, 4, 128).contiguous(), t=b.table[:1].expand(n, -1).contiguous(),
                        n=torch.ones(n, dtype=torch.int32, device=DEV)), "2048")
    # nothing to do
    none = torch.empty(0, 4, 128, dtype=BF, device=DEV)
    assert att(q=none, t=b.table[:0], n=b.seq_lens[:0]).shape == (0, 4, 128)
    assert app(q=none, k=k[:0], v=v[:0], p=pos[:0]).shape == (0, 4, 128)
