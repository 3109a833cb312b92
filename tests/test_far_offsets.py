"""Block-scaled products, quantisation and experts on tensors whose elements lie more than
2^31 and 2^32 elements or bytes behind their first one.  What lies there is compared; the
numbers are such that every sum is exact, or the call's own rows by themselves give the
reference."""

import pytest

torch = pytest.importorskip("torch")

from decodebench_amd import ops  # noqa: E402
from test_moe_wide import reference  # noqa: E402  (the experts, with their roundings counted)

FP8 = torch.float8_e4m3fn
DEV = "cuda"
FAR = 2 ** 32


@pytest.fixture(autouse=True)
def _memory():
    yield
    torch.cuda.empty_cache()


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def small(rows, K, seed):
    """1, 2 and 4 of both signs."""
    g = gen(seed)
    size = torch.randint(0, 3, (rows, K), generator=g, device=DEV).float().exp2()
    return size * (torch.randint(0, 2, (rows, K), generator=g, device=DEV) * 2 - 1)


@pytest.mark.gpu
def test_quantize_far_rows():
    T, K = 2 ** 18 + 5, 16384
    assert T * K > FAR
    x = torch.zeros(T, K, dtype=torch.bfloat16, device=DEV)
    tail = torch.randn(37, K, generator=gen(1), device=DEV).bfloat16()
    x[-37:] = tail
    q, scale = ops.quantize_blocks(x)
    wq, ws = ops.quantize_blocks(tail)
    assert torch.equal(q[-37:].view(torch.uint8), wq.view(torch.uint8))
    assert torch.equal(scale[-37:], ws) and (scale[:-37] == 1).all()
    assert not q[:-37].view(torch.uint8).any()


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 16, 40, 300])
def test_gemm_far_weights(T):
    N, K = 2 ** 19 + 200, 8192
    assert N * K > FAR
    W = torch.zeros(N, K, dtype=torch.uint8, device=DEV).view(FP8)
    some = small(300, K, 2)
    W[-300:] = some.to(FP8)
    ws = torch.ones(-(-N // 128), K // 128, device=DEV)
    ws[-2:] = 0.5
    x = small(T, K, T)
    y = ops.gemm_blocks(x.to(FP8), W, ws, x_scale=torch.full((T, K // 128), 0.125, device=DEV))
    rows = torch.arange(N - 300, N, device=DEV)
    scale = torch.where(rows // 128 >= ws.shape[0] - 2, 0.5, 1.0).double()
    want = (x.double() @ some.double().t()) * 0.125 * scale
    assert torch.equal(y[:, -300:], want.half()) and not y[:, :-300].any()


@pytest.mark.gpu
def test_gemm_far_outputs():
    T, N, K = 8200, 2 ** 19 + 64, 144
    assert T * N > FAR
    W, x = small(N, K, 1), small(T, K, 2)
    one = torch.ones(-(-N // 128), 2, device=DEV)
    y = ops.gemm_blocks(x.to(FP8), W.to(FP8), one, x_scale=torch.ones(T, 2, device=DEV))
    for rows in (slice(0, 3), slice(T - 9, T)):
        assert torch.equal(y[rows], (x[rows].double() @ W.double().t()).half())


@pytest.mark.gpu
def test_route_far_rows():
    T, H, E, k = 2 ** 20 - 3, 4112, 8, 2
    assert T * H > FAR
    x = torch.zeros(T, H, dtype=torch.float16, device=DEV)
    tail = torch.randn(33, H, generator=gen(3), device=DEV).half()
    x[-33:] = tail
    Wr = (torch.randn(E, H, generator=gen(4), device=DEV) / 64).half()
    e, w = ops.moe_route(x, Wr, k)
    te, tw = ops.moe_route(tail, Wr, k)
    assert torch.equal(e[-33:], te) and ((w[-33:] - tw).abs() <= 2.0 ** -22).all()
    assert (e[:-33] == torch.arange(k, device=DEV)).all() and (w[:-33] == 0.5).all()


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 3, 40])
@pytest.mark.parametrize("fp8", [False, True])
def test_far_experts(fp8, T):
    E, H, I, k = (132 if fp8 else 66), 4096, 8208, 2
    assert E * H * I > FAR * (1 if fp8 else 0.5)
    last = [E - 1, E - 2]
    on_gpu, near = {}, {}
    for i, (w, s, shape) in enumerate((("Wg", "sg", (I, H)), ("Wu", "su", (I, H)), ("Wd", "sd", (H, I)))):
        W = torch.zeros(E, *shape, dtype=torch.uint8 if fp8 else torch.float16, device=DEV)
        W = W.view(FP8) if fp8 else W
        for n, e in enumerate(last):
            v = torch.randn(*shape, generator=gen(10 * i + n), device=DEV)
            W[e] = (v * 50).to(FP8) if fp8 else (v / shape[1] ** 0.5).half()
        on_gpu[w], near[w] = W, W[[E - 2, E - 1]].clone() if not fp8 else \
            W.view(torch.uint8)[[E - 2, E - 1]].clone().view(FP8)
        if fp8:
            blocks = (-(-shape[0] // 128), -(-shape[1] // 128))
            on_gpu[s] = torch.ones(E, *blocks, device=DEV)
            on_gpu[s][E - 2:] = 0.02 / shape[1] ** 0.5 * (1 + torch.rand(2, *blocks, generator=gen(9),
                                                                        device=DEV))
            near[s] = on_gpu[s][E - 2:].clone()
    x = torch.randn(T, H, generator=gen(5), device=DEV).half()
    weights = torch.rand(T, k, generator=gen(6), device=DEV)
    ones = torch.tensor([[1, 0]], dtype=torch.int32, device=DEV).repeat(T, 1)
    y = ops.moe_experts(x, ones + (E - 2), weights, **on_gpu)
    # the same two experts by themselves, in 64 bits
    plain = {w: torch.stack([spread(near, w, s, e) for e in range(2)])
             for w, s in (("Wg", "sg"), ("Wu", "su"), ("Wd", "sd"))}
    want, tol = reference(x, ones, weights, plain)
    assert ((y.double() - want).abs() <= tol).all()


def spread(near, w, s, e):
    if s not in near:
        return near[w][e].double()
    W = near[w].view(torch.uint8)[e].view(FP8).double()
    return W * near[s][e].double().repeat_interleave(128, 0)[:W.shape[0]].repeat_interleave(
        128, 1)[:, :W.shape[1]]
