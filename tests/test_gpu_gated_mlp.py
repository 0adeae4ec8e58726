"""GPU parity of ops.gemm_gated_bf16 and ops.gated_mlp against the formulas in
fp64.

Tolerances.  A rounding to bf16 is off by at most 2^-8 of the value.  A product
sum of K exact bf16 products in fp32 is off by at most e = K 2^-23 |x|.|w| (the
tensor core may cut where fp32 would round).  gemm_gated_bf16 rounds once:
2^-8 |o| + 1.13 (e1 |z2| + |act z1| e2 + e1 e2), 1.13 bounding the activations'
slopes, with 2^-20 of |o| for erf and exp.  gated_mlp rounds the inner values
(2^-8 each) and the result, and sums I of them: 2^-8 |o| + T + K 2^-23 (|h| + t).|w3|
with T = (2^-8 |h| + t).|w3|, t the first product's tolerance before rounding."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16


def act64(z, activation):
    if activation == "gelu":
        return 0.5 * z * torch.special.erfc(-z / 2 ** 0.5)
    return z * torch.sigmoid(z) if activation == "silu" else z


def gated64(x, w1, w2, activation):
    """(value, fp32 error bound before rounding)."""
    x, w1, w2 = x.double(), w1.double(), w2.double()
    z1, z2 = x @ w1.T, x @ w2.T
    e1, e2 = (x.shape[1] * 2.0 ** -23 * (x.abs() @ w.abs().T) for w in (w1, w2))
    a = act64(z1, activation)
    return a * z2, 1.13 * (e1 * z2.abs() + a.abs() * e2 + e1 * e2) + 2.0 ** -20 * (a * z2).abs()


def inputs(M, K, N, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    return r(M, K).to(BF), (r(N, K) * K ** -0.5).to(BF), (r(N, K) * K ** -0.5).to(BF)


# rows below, at and beyond a 128-row tile and the SM-pair kernel's switch; K of
# one block, odd numbers of blocks; N of part of a tile, odd numbers of tiles
@pytest.mark.parametrize("M,K,N", [
    (1, 64, 8), (1, 4096, 11008), (7, 192, 72), (3, 128, 22528), (128, 192, 22528), (64, 2048, 5504),
    (90, 512, 30008), (101, 256, 512), (128, 512, 1000), (128, 4096, 11008),
    (129, 320, 136), (300, 512, 2056), (777, 1024, 5504), (4095, 128, 264), (4096, 256, 128),
    (4101, 192, 1160), (5000, 512, 120)])
@pytest.mark.parametrize("activation", ["none", "gelu", "silu"])
def test_gated_gemm(M, K, N, activation):
    from evo2_flash_b200 import ops

    x, w1, w2 = inputs(M, K, N)
    out = ops.gemm_gated_bf16(x, w1, w2, activation)
    ref, t = gated64(x, w1, w2, activation)
    bad = (out.double() - ref).abs() - (2.0 ** -8 * ref.abs() + t)
    assert (bad <= 0).all(), float(bad.max())
    assert torch.equal(ops.gemm_gated_bf16(x, w1, w2, activation), out)
    ops.check_gemm_waits()


@pytest.mark.parametrize("M", [1, 64, 200, 4200])
def test_strides_and_rows_around_are_left(M):
    from evo2_flash_b200 import ops

    K, N = 128, 328
    x, w1, w2 = inputs(M, 2 * K, N, seed=3)
    x, w = x[:, :K], torch.cat([w1, w2], 0)  # views of wider tensors
    room = torch.full((M + 2, N + 24), 3.0, dtype=BF, device=DEV)
    out = room[1:M + 1, 8:8 + N]
    assert ops.gemm_gated_bf16(x, w[:N, K:], w[N:, :K], "gelu", out=out) is out
    ref, t = gated64(x, w[:N, K:], w[N:, :K], "gelu")
    assert ((out.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + t).all()
    edge = torch.ones_like(room, dtype=torch.bool)
    edge[1:M + 1, 8:8 + N] = False
    assert (room[edge] == 3.0).all()


def test_activation_tails_and_nonfinite_rows():
    from evo2_flash_b200 import ops

    x, w1, w2 = inputs(40, 64, 64, seed=5)
    x[:8] *= 200  # |z1| in the hundreds
    x[30] = float("nan")
    for activation in ("none", "gelu", "silu"):
        out = ops.gemm_gated_bf16(x, w1, w2, activation)
        ref, t = gated64(x[:30], w1, w2, activation)
        assert ((out[:30].double() - ref).abs() <= 2.0 ** -8 * ref.abs() + t + 1e-30).all()
        assert torch.isnan(out[30]).all() and torch.isfinite(out[31:]).all()


@pytest.mark.parametrize("M,H,I", [(1, 256, 512), (1, 4096, 11008), (33, 512, 1024), (257, 256, 704),
                                   (4100, 256, 512)])
@pytest.mark.parametrize("activation", ["none", "gelu", "silu"])
def test_gated_mlp(M, H, I, activation):
    from evo2_flash_b200 import ops

    x, w1, w2 = inputs(M, H, I, seed=7)
    w3 = (torch.randn(H, I, device=DEV) * I ** -0.5).to(BF)
    out = ops.gated_mlp(x, w1, w2, w3, activation)
    h, t = gated64(x, w1, w2, activation)
    ref, w = h @ w3.double().T, w3.double().abs().T
    tol = 2.0 ** -8 * ref.abs() + (2.0 ** -8 * h.abs() + t) @ w + I * 2.0 ** -23 * ((h.abs() + t) @ w)
    assert ((out.double() - ref).abs() <= tol).all()
    room = torch.empty(M, H + 8, dtype=BF, device=DEV)[:, :H]
    assert ops.gated_mlp(x, w1, w2, w3, activation, out=room) is room
    assert torch.equal(room, out)


def test_graph_and_streams():
    from evo2_flash_b200 import ops

    x, w1, w2 = inputs(17, 256, 512)
    w3 = (torch.randn(256, 512, device=DEV) * 0.05).to(BF)
    want = ops.gated_mlp(x, w1, w2, w3)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        other = ops.gated_mlp(x, w1, w2, w3)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        held = ops.gated_mlp(x, w1, w2, w3)
    x2 = x.flip(0).contiguous()
    x.copy_(x2)
    g.replay()
    assert torch.equal(other, want) and torch.equal(held, want.flip(0))


def test_refusals():
    from evo2_flash_b200 import ops

    x, w1, w2 = inputs(3, 128, 64)
    w3 = torch.zeros(128, 64, dtype=BF, device=DEV)

    def refused(match, *a, fn=ops.gated_mlp, **kw):
        with pytest.raises(ValueError, match=match):
            fn(*a, **kw)

    refused("bf16", x.float(), w1, w2, w3)
    refused("CUDA", x.cpu(), w1, w2, w3)
    refused("columns", x, w1[:, :64], w2, w3)
    refused("columns", x, w1, w2, w3[:, :32])
    refused("rows", x, w1, w2[:32], w3)
    refused("activation", x, w1, w2, w3, "relu")
    refused("columns", x, w1, w2, w3, out=w3)
    refused("rows", x, w1, w2, w3, out=w3.new_empty(4, 128))
    refused("no backward", x.clone().requires_grad_(), w1, w2, w3)
    refused("multiple of 64", x, w1[:40], w2[:40], w3[:, :40])
    refused("K % 64", x[:, :96], w1[:, :96], w2[:, :96], fn=ops.gemm_gated_bf16)
    refused("N % 8", x, w1[:20], w2[:20], fn=ops.gemm_gated_bf16)
    refused("16-byte", x[:, 1:65], w1[:, :64], w2[:, :64], fn=ops.gemm_gated_bf16)
    assert ops.gated_mlp(x[:0], w1, w2, w3).shape == (0, 128)
