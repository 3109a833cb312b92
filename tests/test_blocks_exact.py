"""``gemm_blocks`` on numbers whose sums are exact: small codes and scales that are
powers of two.

Tolerances that count roundings grow with the rows and cannot see a few columns that a
long row leaves out.  Here every product, every sum in any order and every scaled sum is
a whole number of fp32, far from where the matrix instruction cuts its sums: codes of
1, 2 and 4 have products below 2^5 (2^11 beside one 448 of a block), and K 2^4 times a
spread of scales of 2^3 stays below 2^24.  So the output is the one rounding of the exact
sum, bit for bit, whatever the tile, the parts of K and their order.
"""

import pytest

torch = pytest.importorskip("torch")

from decodebench_amd import ops  # noqa: E402

FP8 = torch.float8_e4m3fn
DEV = "cuda"
TYPES = [torch.float16, torch.bfloat16]


def blocks(n):
    return -(-n // 128)


def small(rows, K, seed):
    """Codes of 1, 2 and 4 of both signs, as fp32."""
    gen = torch.Generator().manual_seed(seed)
    size = torch.randint(0, 3, (rows, K), generator=gen)
    return (torch.exp2(size.float()) * (torch.randint(0, 2, (rows, K), generator=gen) * 2 - 1))


def scales(rows, cols, seed, low, spread):
    gen = torch.Generator().manual_seed(seed)
    return torch.exp2(torch.randint(low, low + spread, (rows, cols), generator=gen).float())


def whole(scale, N, K):
    return scale.double().repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]


def case(T, N, K, seed=0):
    """Inputs on the CPU and the exact sums."""
    q, W = small(T, K, seed + T), small(N, K, seed + N + 1)
    # (sums of fp16 outputs stay below 65504)
    xs, ws = scales(T, blocks(K), seed + 2, -6, 2), scales(blocks(N), blocks(K), seed + 3, -1, 2)
    want = (q.double() * xs.double().repeat_interleave(128, 1)[:, :K]) @ (
        W.double() * whole(ws, N, K)).t()
    return q.to(FP8), xs, W.to(FP8), ws, want


def same(y, want):
    want = want.to(y.device)
    exact = want.float()
    assert torch.equal(exact.double(), want)     # the oracle's own sums are exact in 32 bits
    assert torch.equal(y, exact.to(y.dtype)), f"{(y != exact.to(y.dtype)).sum()} outputs differ"


SIZES = [
    (1, 16, 16), (1, 130, 144), (2, 512, 640), (5, 77, 2064), (16, 256, 1024), (17, 129, 528),
    (48, 384, 4096), (65, 255, 512), (129, 259, 400), (300, 2048, 1536), (1030, 1300, 784),
    # long rows
    (1, 200, 16384), (4, 200, 14336), (16, 200, 14336), (40, 200, 16384), (301, 500, 14336),
    (700, 600, 16384), (9, 8200, 8192),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,N,K", SIZES)
def test_sums_are_exact(dtype, T, N, K):
    q, xs, W, ws, want = case(T, N, K)
    y = ops.gemm_blocks(q.to(DEV), W.to(DEV), ws.to(DEV), x_scale=xs.to(DEV), dtype=dtype)
    same(y, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,N,K", SIZES)
def test_sums_of_rows_quantized_on_the_way_are_exact(dtype, T, N, K):
    """A 448 leads each block, so that its scale is the power of two it was made with."""
    q, xs, W, ws, _ = case(T, N, K)
    q = q.float()
    q[:, ::128] = 448.0 * q[:, ::128].sign()
    x = (q * xs.repeat_interleave(128, 1)[:, :K]).to(dtype)
    want = x.double() @ (W.double() * whole(ws, N, K)).t()
    y = ops.gemm_blocks(x.to(DEV), W.to(DEV), ws.to(DEV))
    same(y, want)


@pytest.fixture
def tuned():
    yield ops.tune
    ops.tune("blocks_shape", 0)
    ops.tune("blocks_parts", 0)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", range(1, 8))
@pytest.mark.parametrize("T,N,K", [(5, 77, 2064), (65, 300, 16384), (200, 1031, 2048),
                                   (300, 520, 14336)])
def test_sums_of_every_tile_shape_are_exact(tuned, shape, T, N, K):
    q, xs, W, ws, want = case(T, N, K, 7)
    args = [t.to(DEV) for t in (q, W, ws)]
    tuned("blocks_shape", shape)
    for parts in (1, 2, 3, 5, 16):
        tuned("blocks_parts", parts)
        same(ops.gemm_blocks(*args, x_scale=xs.to(DEV)), want)


@pytest.mark.parametrize("T,N,K", [(1, 16, 16), (16, 200, 14336), (40, 200, 16384)])
def test_the_oracle_sees_sixteen_columns_left_out(T, N, K):
    q, xs, W, ws, want = case(T, N, K)
    q = q.float()
    q[:, K - 16:] = 0
    less = (q.double() * xs.double().repeat_interleave(128, 1)[:, :K]) @ (
        W.double() * whole(ws, N, K)).t()
    for dtype in TYPES:
        assert (less.to(dtype) != want.to(dtype)).float().mean() > 0.5
