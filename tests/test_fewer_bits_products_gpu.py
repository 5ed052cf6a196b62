"""8-bit products of many tokens against their definition in 64 bits: the kernel on pairs of multiprocessors and the tile of 128 tokens, which
few tokens never reach."""
import math

import pytest
import torch

from test_fewer_bits_gpu import HALF, product, rows_of

pytestmark = pytest.mark.gpu

KINDS = {"bf16": (torch.bfloat16, False, None), "f32": (torch.float32, False, None), "bf16 out32 bias": (torch.bfloat16, True, torch.float32),
         "bf16 bias16": (torch.bfloat16, False, torch.bfloat16), "f32 bias16": (torch.float32, False, torch.bfloat16), "f32 bias": (torch.float32, False, torch.float32)}


def plan(M, N, K, out):
    """The kernel that ``linear`` takes: tokens of a tile, 256 for pairs of multiprocessors."""
    from tinyserve_b200.kernels import ops
    tile, splits = ops.int8_plan(M, N, K)
    return 128 if splits == 0 and N * out.itemsize % 16 else tile


def operands(M, N, K, kind, seed=0):
    dtype, out32, bias = KINDS[kind]
    g = torch.Generator(device="cuda").manual_seed(M + N + K + seed)
    x = (torch.randn(M, K + 5, generator=g, device="cuda") * torch.rand(M, 1, generator=g, device="cuda")).to(dtype)[:, :K]
    b = torch.randn(N, generator=g, device="cuda").to(bias) if bias is not None else None
    return x, rows_of(N, K, seed), b, torch.float32 if out32 else dtype


# (M, N, K, the tile for whole 16-byte rows of output): ragged ends of both sides of a pair's 256 x 256, of K, one and several tiles a pair, one slice of K
SHAPES = [(700, 4096, 2048, 256), (1025, 4616, 1040, 256), (333, 12808, 333, 256), (257, 20480, 128, 256), (129, 38008, 100, 256), (2050, 9000, 300, 256),
          (5000, 520, 1000, 256), (100, 24576, 512, 128), (128, 19000, 1111, 128), (65, 37632, 40, 128), (300, 24571, 500, 128), (2051, 3333, 257, 128), (333, 12812, 777, 256)]


@pytest.mark.parametrize("M,N,K,tile", SHAPES)
@pytest.mark.parametrize("kind", sorted(KINDS))
def test_product_of_many_tokens(M, N, K, tile, kind):
    from tinyserve_b200.kernels import ops
    x, rows, bias, out_type = operands(M, N, K, kind)
    # (the shape still goes where it is meant to go, as long as the device is the one that the rule was measured on)
    if ops.num_sms() == 148:
        assert plan(M, N, K, out_type) == (128 if N * out_type.itemsize % 16 else tile)
    out = ops.linear(x, rows, bias, out_float32=KINDS[kind][1])
    assert out.dtype == out_type
    want, err = product(x, rows, bias)
    assert ((out.double() - want).abs() <= err + HALF[out.dtype] * want.abs() + 1e-30).all()
    again = ops.linear(ops.quantize_rows(x), rows, bias, out_float32=out.dtype == torch.float32, constant_weight=True)
    assert torch.equal(again, out)
    assert ops.gemm_int8_error() == 0


@pytest.mark.parametrize("M,N,K", [(700, 4096, 300), (100, 24576, 200)])
def test_rows_without_a_value_among_many(M, N, K):
    """Rows of zeros, infinities and NaN, on both sides, beside ordinary ones; the largest sums."""
    from tinyserve_b200.kernels import ops
    assert ops.num_sms() != 148 or plan(M, N, K, torch.bfloat16) in (128, 256)
    x, rows, _, _ = operands(M, N, K, "f32")
    x, weights = x.clone(), rows.float()
    x[0], x[M - 1], x[M // 2, 3], x[M // 3, K - 1] = 0, 1, math.nan, -math.inf
    weights[1], weights[N - 1], weights[7, 0], weights[N // 2, 1] = 0, -1, math.inf, math.nan
    rows = ops.quantize_rows(weights)
    out = ops.linear(x, rows)
    bad = torch.zeros(M, N, dtype=torch.bool, device="cuda")
    bad[[M // 2, M // 3]] = True
    bad[:, [7, N // 2]] = True
    assert torch.equal(out.isnan(), bad)
    want, err = product(x, rows)
    assert (((out.double() - want).abs() <= err + HALF[torch.float32] * want.abs() + 1e-30) | bad).all()
    assert not out[0][~bad[0]].any() and not out[:, 1][~bad[:, 1]].any()


@pytest.mark.parametrize("M,N,K", [(700, 4096, 2048), (100, 24576, 512)])
def test_a_captured_product_of_many_tokens_serves_other_inputs(M, N, K):
    from tinyserve_b200.kernels import ops
    x, rows, bias, _ = operands(M, N, K, "bf16 bias16")
    x = x.contiguous()
    ops.linear(x, rows, bias)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.linear(x, rows, bias)
    for seed in range(3):
        x.copy_(torch.randn(M, K, generator=torch.Generator().manual_seed(seed)).bfloat16())
        graph.replay()
        want, err = product(x, rows, bias)
        assert ((out.double() - want).abs() <= err + HALF[out.dtype] * want.abs() + 1e-30).all()
        assert torch.equal(out, ops.linear(x, rows, bias))


@pytest.mark.parametrize("M", [3, 40, 100, 700])
def test_codes_of_a_weight_made_right_before_the_product(M):
    """A weight that is no constant: its codes come from the call before, again and again into the same memory."""
    from tinyserve_b200.kernels import ops
    N, K = 4096, 1024
    g = torch.Generator(device="cuda").manual_seed(M)
    x = torch.randn(M, K, generator=g, device="cuda").bfloat16()
    sources = [torch.randn(N, K, generator=g, device="cuda").bfloat16() for _ in range(4)]
    wants = [product(x, ops.quantize_rows(w)) for w in sources]
    for _ in range(3):
        for w, (want, err) in zip(sources, wants):
            out = ops.linear(x, ops.quantize_rows(w))
            assert ((out.double() - want).abs() <= err + HALF[out.dtype] * want.abs() + 1e-30).all()


@pytest.mark.parametrize("M", [40, 300, 2048])
def test_gated_product_of_many_tokens(M):
    """Gate and up rows in alternating blocks, as feed-forwards hold them: the plain product, then the activation."""
    from tinyserve_b200.kernels import ops
    N, K = 6144, 512
    x, rows, _, _ = operands(M, N, K, "bf16")
    got = ops.gated_linear(x, rows, "silu", block=ops.GATED_BLOCK, constant_weight=True)
    y, err = product(x, rows)
    # (the product is rounded before the activation; silu changes by at most 1.1 of what its argument does)
    y = y.unflatten(1, (-1, 2, ops.GATED_BLOCK))
    gate, up = y[:, :, 0].flatten(1), y[:, :, 1].flatten(1)
    half = HALF[torch.bfloat16]
    off = 2 * half * (1.1 * gate.abs() * up.abs() + (gate * torch.sigmoid(gate) * up).abs())
    assert ((got.double() - gate * torch.sigmoid(gate) * up).abs() <= off + 2.0 ** -20 * gate.abs().max() * up.abs().max()).all()
