"""Cases for the decoder layer's operators beside the Hyena mixers, each in a plain
torch form and, where `own` is true, through this package's kernels:

  append     rotary embedding of a step's queries and keys, with the rotated keys and
             the values written into a paged cache (ops.kv_append)
  attention  a step's queries against the paged cache, the requests of a group
             sharing the leading keys of their prompt (ops.paged_attention)
  mlp        the gated feed-forward block l3(act(x l1^T) * (x l2^T)) (ops.gated_mlp)

Caches are (pages, page size, key/value heads, head dim), stored head by head inside a
page; a request's page table names the page of each run of its positions, and requests
that share a prompt name the same pages.
"""

import math

import torch

own = False

THETA = 10000.0


# ---------------------------------------------------------------- cases
def listed():
    return [
        # One sequence being sampled, one new token: the smallest call there is.
        dict(name="append, one token", op="append", requests=1, new=1, ctx=700, heads=32, kv_heads=32, dim=128,
             page=64, ragged=False),
        # A chunk of a long prompt, far into its context, grouped heads, small pages, odd length.
        dict(name="append, far chunk", op="append", requests=1, new=4099, ctx=126001, heads=32, kv_heads=8, dim=128,
             page=16, ragged=False),
        # The prefill step of the 7B layer shape: eight prompts of 8192 tokens.
        dict(name="append, prefill 64k", op="append", requests=8, new=8192, ctx=0, heads=32, kv_heads=32, dim=128,
             page=64, ragged=False),
        # One sequence being sampled after a short prompt.
        dict(name="attention, one request", op="attention", requests=1, groups=1, new=1, shared=0, kept=777, heads=32,
             kv_heads=32, dim=128, page=64, ragged=False),
        # Independent sequences of very different lengths, nothing shared.
        dict(name="attention, nothing shared", op="attention", requests=32, groups=1, new=1, shared=0, kept=8000,
             heads=32, kv_heads=32, dim=128, page=64, ragged=True),
        # 64 samples of one prompt, each some hundred tokens in.
        dict(name="attention, 64 samples", op="attention", requests=64, groups=1, new=1, shared=8192, kept=500, heads=32,
             kv_heads=32, dim=128, page=64, ragged=True),
        # Speculative verify: four positions a request, three prompts, the shared run ends inside a page.
        dict(name="attention, verify 3 prompts", op="attention", requests=48, groups=3, new=4, shared=2029, kept=700,
             heads=32, kv_heads=32, dim=128, page=16, ragged=True),
        # Many samples of one long prompt, grouped heads.
        dict(name="attention, 256 samples", op="attention", requests=256, groups=1, new=1, shared=32768, kept=1000,
             heads=64, kv_heads=8, dim=128, page=64, ragged=True),
        # The 7B layer's block for one token: the weights are all there is to read.
        dict(name="mlp, one token", op="mlp", rows=1, hidden=4096, inner=11008, act="none"),
        # Layer 0 (with the activation) of a decode step, an odd number of requests.
        dict(name="mlp, decode 101", op="mlp", rows=101, hidden=4096, inner=11008, act="gelu"),
        # The 40B layer's block on a short prompt.
        dict(name="mlp, 40B shape 777", op="mlp", rows=777, hidden=8192, inner=22528, act="none"),
        # A prefill step of the 7B layer's block.
        dict(name="mlp, prefill 8192", op="mlp", rows=8192, hidden=4096, inner=11008, act="none"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["append", "attention", "attention", "mlp"])
    if op == "mlp":
        hidden, inner = rng.choice([(256, 512), (512, 1024), (2048, 5504), (4096, 11008), (8192, 22528)])
        top = 8192 * 4096 * 11008 // (hidden * inner)  # no more products than the largest listed case
        return dict(op=op, rows=_log_int(rng, 1, min(8192, top)), hidden=hidden, inner=inner,
                    act=rng.choice(["none", "gelu", "silu"]))
    heads, kv_heads = rng.choice([(32, 32), (64, 64), (32, 8), (64, 8), (16, 2), (8, 1), (2, 2)])
    dim, page = rng.choice([128, 128, 128, 64]), rng.choice([16, 32, 48, 64, 128, 256])
    ragged = rng.random() < 0.75
    if op == "append":
        requests = _log_int(rng, 1, 256)
        new = 1 if rng.random() < 0.4 else _log_int(rng, 1, max(1, 65536 * 32 // heads // requests))
        keys = (1 << 28) // (kv_heads * dim * requests)  # 0.5 GB for keys, as much for values
        return dict(op=op, requests=requests, new=new, ctx=_log_int(rng, 1, max(2, min(126000, keys - new))) - 1,
                    heads=heads, kv_heads=kv_heads, dim=dim, page=page, ragged=ragged)
    new = rng.choice([1, 1, 1, 2, 4, 8])
    groups = rng.choice([1, 1, 2, 3, 5])
    requests = groups * _log_int(rng, 1, 256 // groups)
    work = 256 * 64 * 33000 // (requests * new * heads)  # keys a query may see: no more than the largest listed case
    shared = 0 if rng.random() < 0.25 else _log_int(rng, 1, min(32768, work, (1 << 27) // (groups * kv_heads * dim)))
    # the plain form widens every request's own keys to 32 bits, padded to the longest
    kept = _log_int(rng, new, max(new, min(8192, (1 << 29) // (requests * kv_heads * dim))))
    return dict(op=op, requests=requests, groups=groups, new=new, shared=shared, kept=kept, heads=heads,
                kv_heads=kv_heads, dim=dim, page=page, ragged=ragged)


def _spread(n, lo, hi, ragged):
    """n lengths in [lo, hi], fixed by the case alone; all hi when not ragged."""
    if not ragged:
        return [hi] * n
    return [lo + (hi - lo) * ((i * 7919 + 613) % 1009) // 1008 for i in range(n)]


def _sizes(c):
    """Per request: positions already in the cache that only it has, and new tokens."""
    n = c["requests"]
    if c["op"] == "append":
        return _spread(n, 0, c["ctx"], c["ragged"]), _spread(n, 1, c["new"], c["ragged"])
    kept = _spread(n, c["new"], max(c["new"], c["kept"]), c["ragged"])  # new tokens included
    return kept, [c["new"]] * n


# ---------------------------------------------------------------- inputs
def _normal(gen, *shape, scale=1.0):
    t = torch.empty(*shape, dtype=torch.bfloat16, device="cuda").normal_(generator=gen)
    return t.mul_(scale) if scale != 1.0 else t


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _cache(gen, pages, c):
    """(pages, page, kv heads, dim), the heads of a page one after the other in memory."""
    return _normal(gen, pages, c["kv_heads"], c["page"], c["dim"]).transpose(1, 2)


def _inputs(c, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if c["op"] == "mlp":
        h, i = c["hidden"], c["inner"]
        return dict(x=_normal(gen, c["rows"], h), w1=_normal(gen, i, h, scale=0.02),
                    w2=_normal(gen, i, h, scale=0.02), w3=_normal(gen, h, i, scale=0.02))
    n, page = c["requests"], c["page"]
    before, new = _sizes(c)
    heads, kv_heads, dim = c["heads"], c["kv_heads"], c["dim"]
    starts = [0]
    for m in new:
        starts.append(starts[-1] + m)
    tokens = starts[-1]
    order = torch.Generator().manual_seed(seed)
    if c["op"] == "append":
        total = [b + m for b, m in zip(before, new)]
        width = max(-(-t // page) for t in total)
        pages = sum(-(-t // page) for t in total)
        ids = torch.randperm(pages, generator=order).tolist()
        table, at = [], 0
        for t in total:
            m = -(-t // page)
            table.append(ids[at:at + m] + [0] * (width - m))
            at += m
        qkv = _normal(gen, tokens, (heads + 2 * kv_heads) * dim)  # the projection's output, one row a token
        q, k, v = qkv.split([heads * dim, kv_heads * dim, kv_heads * dim], dim=1)
        positions = torch.cat([torch.arange(b, b + m) for b, m in zip(before, new)])
        return dict(q=q.view(tokens, heads, dim), k=k.view(tokens, kv_heads, dim), v=v.view(tokens, kv_heads, dim),
                    positions=positions.to("cuda", torch.int32), starts=_ints(starts), table=_ints(table),
                    k_cache=_cache(gen, pages, c), v_cache=_cache(gen, pages, c))
    shared, groups = c["shared"], c["groups"]
    members = n // groups
    whole = shared // page  # pages that every member of a group names
    width = max(-(-(shared + b) // page) for b in before)
    pages = groups * whole + sum(-(-(shared + b) // page) - whole for b in before)
    ids = torch.randperm(pages, generator=order).tolist()
    table, at = [], groups * whole
    for r, b in enumerate(before):
        g, m = r // members, -(-(shared + b) // page) - whole
        table.append(ids[g * whole:(g + 1) * whole] + ids[at:at + m] + [0] * (width - whole - m))
        at += m
    k_cache, v_cache = _cache(gen, pages, c), _cache(gen, pages, c)
    if shared % page:  # each member has its own copy of the page in which the shared run ends
        ends = torch.tensor([row[whole] for row in table], device="cuda")
        first = ends.view(groups, members)[:, :1].expand(groups, members).reshape(-1)
        for cache in (k_cache, v_cache):
            cache[ends, :shared % page] = cache[first, :shared % page]
    return dict(q=_normal(gen, tokens, heads, dim), k_cache=k_cache, v_cache=v_cache, table=_ints(table),
                seq_lens=_ints([shared + b for b in before]), shared_lens=_ints([shared] * groups),
                group_start=_ints([g * members for g in range(groups + 1)]), starts=_ints(starts))


def prepare(case, seed):
    return dict(_inputs(case, seed), case=case)


# ---------------------------------------------------------------- plain forms
def _plain_append(s):
    c = s["case"]
    half = c["dim"] // 2
    # angles in 64 bits: at position 100000 a 32-bit one is off by hundredths
    inv = THETA ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
    angle = s["positions"].double()[:, None] * inv
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def rotate(x):
        a, b = x[..., :half].float(), x[..., half:].float()
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1).to(x.dtype)

    row = torch.arange(s["positions"].numel(), device="cuda", dtype=torch.int32)
    request = (row[:, None] >= s["starts"][None, 1:]).sum(1)
    pos = s["positions"].long()
    page = s["table"][request, pos // c["page"]].long()
    q = rotate(s["q"])
    s["k_cache"][page, pos % c["page"]] = rotate(s["k"])
    s["v_cache"][page, pos % c["page"]] = s["v"]
    return [q, s["k_cache"], s["v_cache"]]


def _gather(cache, table, at, page):
    """(rows, kv heads, keys, dim) in 32 bits: the cache's rows at positions `at` of each row of `table`."""
    return cache[table.long().gather(1, at // page), at % page].transpose(1, 2).float()


def _plain_attention(s):
    c = s["case"]
    n, groups, new, shared = c["requests"], c["groups"], c["new"], c["shared"]
    hkv, per, dim, page = c["kv_heads"], c["heads"] // c["kv_heads"], c["dim"], c["page"]
    members = n // groups
    q = s["q"].float() * dim ** -0.5
    # the requests' own keys, padded to the longest: (n, kv heads, new * per, keys)
    own_len = s["seq_lens"].long() - shared
    width = max(_sizes(c)[0])
    j = torch.arange(width, device="cuda")
    at = (shared + j).expand(n, width).clamp(max=s["table"].shape[1] * page - 1)
    k2, v2 = _gather(s["k_cache"], s["table"], at, page), _gather(s["v_cache"], s["table"], at, page)
    q2 = q.view(n, new, hkv, per, dim).permute(0, 2, 1, 3, 4).reshape(n, hkv, new * per, dim)
    s2 = (q2 @ k2.transpose(2, 3)).view(n, hkv, new, per, width)
    last = own_len[:, None] - new + torch.arange(new, device="cuda")  # the last own key each query sees
    s2 = torch.where(j > last[:, None, :, None, None], -math.inf, s2)
    # the shared keys, once for each group: (groups, kv heads, members * new * per, keys)
    at = torch.arange(shared, device="cuda").expand(groups, shared)
    first = s["table"][::members]
    k1, v1 = _gather(s["k_cache"], first, at, page), _gather(s["v_cache"], first, at, page)
    q1 = q.view(groups, members * new, hkv, per, dim).permute(0, 2, 1, 3, 4).reshape(groups, hkv, members * new * per, dim)
    s1 = (q1 @ k1.transpose(2, 3)).view(groups, hkv, members, new, per, shared)
    s1 = s1.transpose(1, 2).reshape(n, hkv, new, per, shared)
    top = torch.cat([s1.amax(-1, keepdim=True), s2.amax(-1, keepdim=True)], -1).amax(-1, keepdim=True) if shared \
        else s2.amax(-1, keepdim=True)
    p1, p2 = (s1 - top).exp(), (s2 - top).exp()
    total = p1.sum(-1, keepdim=True) + p2.sum(-1, keepdim=True)
    o2 = (p2.view(n, hkv, new * per, width) @ v2).view(n, hkv, new, per, dim)
    p1 = p1.view(groups, members, hkv, new, per, shared).transpose(1, 2).reshape(groups, hkv, members * new * per, shared)
    o1 = (p1 @ v1).view(groups, hkv, members, new, per, dim).transpose(1, 2).reshape(n, hkv, new, per, dim)
    o = ((o1 + o2) / total).transpose(1, 2).reshape(n * new, hkv * per, dim)
    return o.to(s["q"].dtype)


def _plain_mlp(s):
    x = s["x"].float()
    z, act = x @ s["w1"].float().t(), s["case"]["act"]
    if act == "gelu":
        z = z * 0.5 * (1.0 + torch.erf(z * 0.5 ** 0.5))
    elif act == "silu":
        z = z / (1.0 + (-z).exp())
    return ((z * (x @ s["w2"].float().t())) @ s["w3"].float().t()).to(s["x"].dtype)


# ---------------------------------------------------------------- one pass
def run(s):
    c = s["case"]
    if own:
        from evo2_flash_b200 import ops

        if c["op"] == "append":
            starts = None if c["new"] == 1 else s["starts"]
            q = ops.kv_append(s["q"], s["k"], s["v"], s["positions"], s["k_cache"], s["v_cache"], s["table"],
                              query_start_loc=starts, rope_theta=THETA)
            return [q, s["k_cache"], s["v_cache"]]
        if c["op"] == "attention":
            more = dict(query_start_loc=s["starts"]) if c["new"] > 1 else {}
            if c["shared"]:
                more.update(shared_lens=s["shared_lens"], group_start=s["group_start"])
            return ops.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["seq_lens"], **more)
        return ops.gated_mlp(s["x"], s["w1"], s["w2"], s["w3"], activation=c["act"])
    return {"append": _plain_append, "attention": _plain_attention, "mlp": _plain_mlp}[c["op"]](s)


def work(c):
    if c["op"] == "mlp":
        m, h, i = c["rows"], c["hidden"], c["inner"]
        return dict(bytes=2 * (3 * h * i + 2 * m * h), flops=6 * m * h * i)
    before, new = _sizes(c)
    heads, kv_heads, dim = c["heads"], c["kv_heads"], c["dim"]
    tokens = sum(new)
    if c["op"] == "append":
        # q, k, v read and written, a position and a page each
        return dict(bytes=tokens * (4 * dim * (heads + 2 * kv_heads) + 8), flops=3 * tokens * dim * (heads + kv_heads))
    shared, groups = c["shared"], c["groups"]
    keys = groups * shared + sum(before)
    seen = sum(m * shared + m * b - m * (m - 1) // 2 for b, m in zip(before, new))
    return dict(bytes=4 * keys * kv_heads * dim + 4 * tokens * heads * dim + 4 * (keys // c["page"] + len(before)),
                flops=4 * seen * heads * dim)


# ---------------------------------------------------------------- from the definitions, in 64 bits
def exact(case, seed):
    c, s = case, _inputs(case, seed)
    if c["op"] == "mlp":
        x, w1, w2, w3 = (s[k].double() for k in ("x", "w1", "w2", "w3"))
        z = torch.matmul(x, w1.mT)
        if c["act"] == "gelu":
            z = z * torch.special.erfc(-z / math.sqrt(2.0)) / 2.0
        elif c["act"] == "silu":
            z = z * torch.sigmoid(z)
        return torch.matmul(z.mul(torch.matmul(x, w2.mT)), w3.mT)
    before, new = _sizes(c)
    page, dim = c["page"], c["dim"]
    if c["op"] == "append":
        # a pair (x[i], x[i + dim / 2]) is a complex number, turned by exp(i angle)
        freq = torch.tensor([THETA ** (-2.0 * i / dim) for i in range(dim // 2)], dtype=torch.float64, device="cuda")
        turn = torch.exp(1j * s["positions"].double()[:, None, None] * freq)

        def rotate(x):
            z = torch.complex(x[..., :dim // 2].double(), x[..., dim // 2:].double()) * turn
            return torch.cat([z.real, z.imag], -1)

        q, k, v = rotate(s["q"]), rotate(s["k"]), s["v"].double()
        caches = [s["k_cache"].double(), s["v_cache"].double()]
        at = 0
        for r, (b, m) in enumerate(zip(before, new)):
            pos = torch.arange(b, b + m, device="cuda")
            where = s["table"][r].long()[pos // page]
            for cache, rows in zip(caches, (k, v)):
                cache[where, pos % page] = rows[at:at + m]
            at += m
        return [q, *caches]
    per = c["heads"] // c["kv_heads"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    at = 0
    for r, (b, m) in enumerate(zip(before, new)):
        length = c["shared"] + b
        used = s["table"][r, :-(-length // page)].long()
        k, v = (t[used].reshape(-1, c["kv_heads"], dim)[:length].double() for t in (s["k_cache"], s["v_cache"]))
        q = s["q"][at:at + m].double().unflatten(1, (c["kv_heads"], per))
        scores = torch.einsum("thpd,khd->thpk", q, k) / math.sqrt(dim)
        seen = torch.arange(length, device="cuda") <= length - m + torch.arange(m, device="cuda")[:, None]
        w = torch.softmax(scores.masked_fill(~seen[:, None, None], -math.inf), -1)
        out[at:at + m] = torch.einsum("thpk,khd->thpd", w, v).flatten(1, 2)
        at += m
    return out
