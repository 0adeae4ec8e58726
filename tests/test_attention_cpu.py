"""Host-side refusals of the attention-cache and gated-GEMM entry points, straight
at the C ABI: each returns before anything is launched, so no GPU is needed (the
pointers are never dereferenced)."""

import ctypes as C

import pytest


@pytest.fixture(scope="module")
def lib():
    from evo2_flash_b200 import _build, _lib

    _build.build()
    return _lib.load()


def cache(kv):
    kv.k = kv.v = kv.page_table = 4096
    kv.k_page_stride = kv.v_page_stride = 2 * 16 * 128
    kv.k_token_stride = kv.v_token_stride = 128
    kv.k_head_stride = kv.v_head_stride = 16 * 128
    kv.page_table_stride = kv.pages_per_request = 4
    kv.num_pages, kv.page_size, kv.kv_heads, kv.head_dim = 9, 16, 2, 128


def append_args(**change):
    from evo2_flash_b200._lib import KvAppendArgs

    a = KvAppendArgs()
    cache(a.kv)
    a.q = a.q_out = a.k = a.v = a.positions = 4096
    for n in ("q", "q_out", "k", "v"):
        setattr(a, n + "_token_stride", 512)
        setattr(a, n + "_head_stride", 128)
    a.T, a.num_requests, a.heads, a.rope_theta = 3, 3, 4, 1e4
    return changed(a, change)


def attention_args(**change):
    from evo2_flash_b200._lib import PagedAttentionArgs

    a = PagedAttentionArgs()
    cache(a.kv)
    a.q = a.out = a.seq_lens = 4096
    a.q_token_stride = a.out_token_stride = 512
    a.q_head_stride = a.out_head_stride = 128
    a.T, a.num_requests, a.heads, a.scale = 3, 3, 4, 0.1
    return changed(a, change)


def changed(a, change):
    for k, v in change.items():
        setattr(a.kv if k.startswith("kv_") and hasattr(a.kv, k[3:]) else a,
                k[3:] if k.startswith("kv_") and hasattr(a.kv, k[3:]) else k, v)
    return a


CACHE_REFUSALS = [
    ({"kv_k": None}, b"null"), ({"kv_page_table": None}, b"null"), ({"kv_v": 4100}, b"aligned"),
    ({"kv_k_token_stride": 100}, b"multiples of 8"), ({"kv_page_size": 24}, b"multiple of 16"),
    ({"kv_page_size": 0}, b"multiple of 16"), ({"kv_num_pages": 0}, b"no pages"),
    ({"kv_pages_per_request": 0}, b"no pages"), ({"kv_head_dim": 96}, b"64 or 128"),
    ({"kv_pages_per_request": 1 << 28}, b"2^31"), ({"kv_kv_heads": 0}, b"kv_heads"),
]


@pytest.mark.parametrize("change,text", CACHE_REFUSALS + [
    ({"T": -1}, b"negative"), ({"k": None}, b"null"), ({"positions": None}, b"null"),
    ({"q_out": None}, b"go together"), ({"heads": 0}, b"heads"), ({"v": 4104}, b"aligned"),
    ({"q_head_stride": 4}, b"multiples of 8"), ({"rope_theta": -1.0}, b"rope_theta"),
    ({"rope_theta": float("inf")}, b"rope_theta"),
])
def test_append_refuses(lib, change, text):
    a = append_args(**change)
    assert lib.hyena_kv_append(C.byref(a), None) == 1
    assert text in lib.hyena_last_error()


@pytest.mark.parametrize("change,text", CACHE_REFUSALS + [
    ({"num_requests": -1}, b"negative"), ({"q": None}, b"null"), ({"seq_lens": None}, b"null"),
    ({"heads": 3}, b"multiple of kv_heads"), ({"out": 4104}, b"aligned"),
    ({"out_token_stride": 4}, b"multiples of 8"), ({"num_groups": 1}, b"go together"),
    ({"shared_lens": 4096}, b"go together"), ({"shared_lens": 4096, "num_groups": 2}, b"group_start"),
    ({"T": 2100, "num_requests": 2100}, b"2048"), ({"T": 1 << 30}, b"too many"),
    ({"scale": float("nan")}, b"finite"), ({"scale": float("inf")}, b"finite"),
    ({}, b"workspace"),  # several chunks fit the table: a workspace is needed
])
def test_attention_refuses(lib, change, text):
    a = attention_args(**{"kv_pages_per_request": 64, **change})
    assert lib.hyena_paged_attention(C.byref(a), None, 0, None) == 1
    assert text in lib.hyena_last_error()


def test_null_arguments_and_empty_steps(lib):
    assert lib.hyena_kv_append(None, None) == 1
    assert lib.hyena_paged_attention(None, None, 0, None) == 1
    assert lib.hyena_paged_attention_workspace_size(None) == 0
    for a in (append_args(T=0), append_args(num_requests=0)):
        assert lib.hyena_kv_append(C.byref(a), None) == 0
    for a in (attention_args(T=0), attention_args(num_requests=0)):
        assert lib.hyena_paged_attention(C.byref(a), None, 0, None) == 0
        assert lib.hyena_paged_attention_workspace_size(C.byref(a)) == 0


def test_workspace_is_bounded(lib):
    """The plan, and a few pieces a row: at most what the pages hold, and 256 MB
    beyond the plan while one piece a row allows it."""
    size = lambda **kw: lib.hyena_paged_attention_workspace_size(C.byref(attention_args(**kw)))  # noqa: E731
    assert size(kv_pages_per_request=8) == 256 + 3 * 4 * 4 * 130 * 4  # 128 keys: four pieces a row
    assert size(kv_pages_per_request=1, shared_lens=4096, num_groups=1) == 256 + 3 * 4 * 2 * 130 * 4
    assert size(kv_pages_per_request=1) == 256 + 3 * 4 * 130 * 4
    for T in (1, 64, 1024):
        assert 0 < size(T=T, num_requests=T, heads=64, kv_pages_per_request=1 << 16) <= (256 << 20) + 16384


@pytest.mark.parametrize("change,text", [
    (dict(act=3), b"activation"), (dict(K=96), b"K % 64"), (dict(N=12), b"N % 8"), (dict(A=4104), b"aligned"),
    (dict(ldb2=60), b"16 bytes"), (dict(ldb1=64), b"too small"), (dict(ldo=16), b"too small"),
    (dict(B2=None), b"null"),
])
def test_gated_gemm_refuses(lib, change, text):
    a = dict(A=4096, lda=128, B1=4096, ldb1=128, B2=4096, ldb2=128, out=4096, ldo=64, M=3, N=64, K=128, act=0)
    a.update(change)
    assert lib.hyena_gemm_gated_bf16(*a.values(), None) == 1
    assert text in lib.hyena_last_error()


def test_packed_arguments_have_the_structs_layout():
    """ops.py packs the argument structs itself: every field lands where the C
    struct (the ctypes declaration) has it."""
    from evo2_flash_b200 import ops
    from evo2_flash_b200._lib import KvAppendArgs, PagedAttentionArgs

    def flat(s):
        for name, kind in s._fields_:
            v = getattr(s, name)
            if isinstance(v, C.Structure):
                yield from flat(v)
            else:
                yield v or 0

    def fill(s, n=1):
        for name, kind in s._fields_:
            if issubclass(kind, C.Structure):
                n = fill(getattr(s, name), n)
            else:
                setattr(s, name, n)
                n += 1
        return n

    for kind, packed in ((KvAppendArgs, ops._KV_APPEND), (PagedAttentionArgs, ops._PAGED_ATTENTION)):
        a = kind()
        fill(a)
        values = list(flat(a))
        assert packed.size <= C.sizeof(kind)  # the struct may end in padding
        b = kind.from_buffer_copy(packed.pack(*values).ljust(C.sizeof(kind), b"\0"))
        assert list(flat(b)) == values
