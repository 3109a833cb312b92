"""Mixture-of-experts layers at the widths of models, and on numbers at the ends of
their types' ranges, against plain forms in 64 bits.

Small layers leave the kernels' loops after one turn.  Here a wave of the kernels for
a few tokens has several rows, several items of a row, and more of h than its first
loads hold; the tiles of eight waves have several slices of rows, and refill every
stage of K.

Tolerances count roundings, u being half a step of the activations' type (fp16 2^-11,
bf16 2^-8): with Sg = sum |Wg x| of a row, g and u are off by (H + 2) 2^-23 Sg and Su
(block scales included), silu by at most 1.1 times that and 2^-21 of itself, h by its
rounding u |h| (for fp16 2^-25 where it is below 2^-14) on top; the down product adds
(I + 2) 2^-23 of the sum of magnitudes, the weights and their sum 2^-22 and k 2^-23,
the output u |y| (2^-25 for fp16).
"""

import pytest

torch = pytest.importorskip("torch")

from decodebench_amd import ops, quant  # noqa: E402

HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
LOWEST = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}
DEV = "cuda"
TYPES = [torch.float16, torch.bfloat16]


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def normal(shape, seed, std=1.0):
    return torch.randn(*shape, generator=gen(seed), device=DEV) * std


def layer(E, H, I, dtype, fp8, seed, std=(None, None)):
    """(weights as the ops take them, the same in 64 bits); std of gate and up, of down
    (not given: one over the root of a row's length)."""
    on_gpu, plain = {}, {}
    for n, (w, s, shape, size) in enumerate((("Wg", "sg", (E, I, H), std[0]),
                                             ("Wu", "su", (E, I, H), std[0]),
                                             ("Wd", "sd", (E, H, I), std[1]))):
        W = normal(shape, 3 * seed + n, size or shape[-1] ** -0.5)
        if fp8:
            on_gpu[w], on_gpu[s] = quant.quantize_e4m3_blocks(W)
            step = on_gpu[s].double().repeat_interleave(128, 1)[:, :shape[1]]
            plain[w] = on_gpu[w].double() * step.repeat_interleave(128, 2)[..., :shape[2]]
        else:
            top = torch.finfo(dtype).max
            on_gpu[w] = W.clamp(-top, top).to(dtype)
            plain[w] = on_gpu[w].double()
    return on_gpu, plain


def reference(x, experts, weights, plain, rounded=True):
    """(y, tolerance) in 64 bits, an expert's tokens at a time; ``rounded``: with that of h."""
    u, low = HALF_STEP[x.dtype], LOWEST[x.dtype]
    x, k = x.double(), experts.shape[1]
    E, I, H = plain["Wg"].shape
    y, tol = torch.zeros_like(x), torch.zeros_like(x)
    for e in range(E):
        t, j = torch.nonzero(experts == e, as_tuple=True)
        if t.numel() == 0:
            continue
        Wg, Wu, Wd = (plain[n][e] for n in ("Wg", "Wu", "Wd"))
        share = weights[t, j].double()[:, None]
        g, up = x[t] @ Wg.t(), x[t] @ Wu.t()
        eg = (H + 2) * 2.0 ** -23 * (x[t].abs() @ Wg.abs().t())
        eu = (H + 2) * 2.0 ** -23 * (x[t].abs() @ Wu.abs().t())
        silu = g / (1 + torch.exp(-g))
        h = silu * up
        es = 1.1 * eg + 2.0 ** -21 * silu.abs()
        eh = es * up.abs() + silu.abs() * eu + es * eu
        if rounded:
            eh = eh + u * (h.abs() + eh) + low
        size = h.abs() @ Wd.abs().t()
        y.index_add_(0, t, share * (h @ Wd.t()))
        tol.index_add_(0, t, share.abs() * (eh @ Wd.abs().t() * 1.01
                                            + ((I + 2 + k) * 2.0 ** -23 + 2.0 ** -22) * size))
    return y, tol + u * (y.abs() + tol) + low


def near(y, want, tol):
    off = (y.double() - want).abs()
    assert (off <= tol).all(), f"{(off / tol).nan_to_num(1e9).max()} of the tolerance"


def routed(T, E, k, seed):
    order = torch.rand(T, E, generator=gen(seed), device=DEV).argsort(1)
    return (order[:, :k].int().contiguous(),
            torch.rand(T, k, generator=gen(seed + 1), device=DEV))


def check(T, E, k, H, I, dtype, fp8):
    on_gpu, plain = layer(E, H, I, dtype, fp8, T + H)
    x = normal((T, H), 5).to(dtype)
    experts, weights = routed(T, E, k, I)
    near(ops.moe_experts(x, experts, weights, **on_gpu), *reference(x, experts, weights, plain))
    # the whole layer: as in two calls
    Wr = normal((E, H), 9, H ** -0.5).to(dtype)
    e, w = ops.moe_route(x, Wr, k)
    y = ops.moe_layer(x, Wr, top_k=k, **on_gpu)
    assert torch.equal(y, ops.moe_experts(x, e, w, **on_gpu))
    near(y, *reference(x, e, w, plain))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("T,E,k,H,I", [
    # several rows a wave, items of a row, a last one in part
    (1, 2, 2, 4112, 2064), (4, 4, 1, 2576, 144), (2, 3, 2, 5136, 2064), (3, 4, 2, 2064, 4112),
    # more of h than the first loads hold
    (1, 2, 2, 144, 14336), (1, 8, 8, 2064, 1040), (4, 8, 8, 1040, 2064),
    # a layer of large experts; of small ones, beyond a launch's tiles of few tokens
    (1, 2, 2, 4096, 14336), (2, 4, 2, 4096, 14336), (9, 4, 2, 4112, 2064),
    # tiles of eight waves: slices of rows, stages in turn
    (150, 2, 1, 1168, 1040), (140, 2, 2, 656, 1296), (300, 3, 1, 1040, 2064), (67, 2, 2, 528, 784),
])
def test_layers_of_models_widths(dtype, fp8, T, E, k, H, I):
    check(T, E, k, H, I, dtype, fp8)


# x and the weights, as powers of two: what g comes to is near one.
RANGES = {
    (torch.float16, "subnormal x"): (-18, 13.5), (torch.float16, "subnormal weights"): (13, -17.5),
    (torch.bfloat16, "subnormal x"): (-130, 125.5),
    (torch.bfloat16, "subnormal weights"): (125, -129.5),
    (torch.bfloat16, "large x"): (100, -104.5),
}


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 4, 24, 200])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dtype,what", list(RANGES))
def test_experts_at_the_ends_of_the_range(dtype, what, fp8, T):
    E, k, H, I = 3, 2, 512, 272
    size, weight = (2.0 ** n for n in RANGES[dtype, what])
    # (scales of subnormal weights would be below fp32's normal numbers)
    if fp8 and "weights" in what and dtype == torch.bfloat16:
        weight, size = 2.0 ** -115.5, 2.0 ** 111
    on_gpu, plain = layer(E, H, I, dtype, fp8, T, (weight, None))
    x = normal((T, H), 7, size).to(dtype)
    assert x.isfinite().all()
    experts, weights = routed(T, E, k, 3)
    near(ops.moe_experts(x, experts, weights, **on_gpu), *reference(x, experts, weights, plain))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("T,E,k,H,I", [(1, 4, 2, 512, 272), (4, 4, 2, 272, 528), (1, 2, 2, 256, 14336),
                                       (2, 4, 4, 256, 6160)])
def test_few_tokens_keep_h_in_32_bits(dtype, fp8, T, E, k, H, I):
    """h is near 2^18, which fp16 does not hold, and a layer is off by less than a rounding
    of h alone would cost: the steps of all other roundings are counted, that one not."""
    on_gpu, plain = layer(E, H, I, dtype, fp8, T, (2.0 ** 9 / H ** 0.5, 2.0 ** -17 / I ** 0.5))
    x = normal((T, H), 7).to(dtype)
    experts, weights = routed(T, E, k, 3)
    weights += 0.5
    y = ops.moe_experts(x, experts, weights, **on_gpu)
    want, tol = reference(x, experts, weights, plain, rounded=False)
    near(y, want, tol)
    # The output's rounding is off by up to u 2^e, u 2^e / sqrt(3) in the root mean square:
    # 0.41 u of normally distributed outputs.  One of h as well would make that 0.58 u.
    off = (y.double() - want).square().mean().sqrt() / want.square().mean().sqrt()
    assert off <= 0.5 * HALF_STEP[dtype]


@pytest.mark.gpu
@pytest.mark.parametrize("T", [5, 24, 200])
def test_tokens_whose_h_leaves_fp16_stay_alone(T):
    """In calls of more than a few tokens, whose h is rounded to fp16."""
    E, k, H, I = 3, 2, 512, 272
    on_gpu, _ = layer(E, H, I, torch.float16, False, T, (2.0 ** 3 / H ** 0.5, 2.0 ** -8 / I ** 0.5))
    x = normal((T, H), 7).half()
    experts, weights = routed(T, E, k, 3)
    clean = ops.moe_experts(x, experts, weights, **on_gpu)
    assert clean.isfinite().all()
    x[T // 2] *= 2.0 ** 8
    y = ops.moe_experts(x, experts, weights, **on_gpu)
    keep = torch.arange(T, device=DEV) != T // 2
    assert torch.equal(y[keep], clean[keep]) and not y[T // 2].isfinite().any()


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 4, 24, 200])
@pytest.mark.parametrize("fp8", [False, True])
def test_experts_whose_h_is_subnormal(fp8, T):
    """h near 2^-19 in fp16, down weights that bring it back to one."""
    E, k, H, I = 3, 2, 512, 272
    on_gpu, plain = layer(E, H, I, torch.float16, fp8, T, (2.0 ** -13.5, 2.0 ** 12))
    x = normal((T, H), 7).half()
    experts, weights = routed(T, E, k, 3)
    near(ops.moe_experts(x, experts, weights, **on_gpu), *reference(x, experts, weights, plain))
