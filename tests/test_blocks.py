"""Block-scaled e4m3: ``quantize_blocks`` and ``gemm_blocks`` against plain
implementations in 64 bits, their refusals, and a product after a quantisation.

Tolerances count roundings: u is half a step of the output's type (fp16 2^-11,
bf16 2^-8).

* quantize_blocks: none.  The scale is an fp32 product of a 16-bit magnitude and the
  rounded 1 / 448, which 64 bits hold exactly; the codes are e4m3 of an fp32
  quotient, and a quotient in 64 bits rounded to 32 is the same number.
* gemm_blocks: products of e4m3 are exact; with S = sum_k |x_k W_k| (scales
  included) K fp32 additions are off by at most 2^-23 S each, also where they cut
  instead of rounding, the scales and their products by 2^-22 S in all, the
  output by u |y|:  u |y| + (K + 2) 2^-23 S.
"""

import ctypes as C

import pytest

torch = pytest.importorskip("torch")

from decodebench_amd import ops, quant  # noqa: E402

HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
FP8 = torch.float8_e4m3fn
DEV = "cuda"
TYPES = [torch.float16, torch.bfloat16]


def blocks(n):
    return -(-n // 128)


def generator(seed):
    return torch.Generator().manual_seed(seed)


def quantized(x):
    """The definition, block after block, on the CPU: (q, scale)."""
    x = x.cpu()
    T, K = x.shape
    q = torch.empty(T, K, dtype=FP8)
    scale = torch.empty(T, blocks(K), dtype=torch.float32)
    for b in range(blocks(K)):
        part = x[:, 128 * b:128 * b + 128].double()
        s = (part.abs().amax(1) * torch.tensor(1.0 / 448.0).double()).float()
        s[s == 0] = 1.0
        v = (part / s.double()[:, None]).float().clamp(-448.0, 448.0)
        q[:, 128 * b:128 * b + 128] = v.to(FP8)
        scale[:, b] = s
    return q, scale


def same_codes(got, want):
    g, w = got.cpu().float(), want.float()
    return torch.equal(g.isnan(), w.isnan()) and torch.equal(g.nan_to_num(), w.nan_to_num())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,K", [(1, 16), (1, 4096), (3, 144), (16, 512), (17, 528), (33, 2064),
                                 (300, 1040), (1, 14336)])
def test_quantize(dtype, T, K):
    x = (torch.randn(T, K, generator=generator(T + K)) * 3).to(dtype)
    x[0, :16] *= 100
    q, scale = ops.quantize_blocks(x.to(DEV))
    wq, ws = quantized(x)
    assert q.dtype == FP8 and q.shape == (T, K) and q.is_contiguous()
    assert scale.shape == (T, blocks(K)) and scale.dtype == torch.float32
    assert torch.equal(scale.cpu(), ws)
    assert same_codes(q, wq)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_values_on_and_beside_borders(dtype):
    """Every magnitude of the type against several scales: ties between two codes,
    the smallest numbers, the largest, numbers that scale to less than a step."""
    bits = torch.arange(0x7C00 if dtype == torch.float16 else 0x7F80, dtype=torch.int32)
    every = bits.to(torch.int16).view(dtype)
    rows = []
    for top in (1.0, 448.0, 7.0, 0.1, 3e-5, 60000.0):
        # chunks of 127 magnitudes below the block's largest, which leads it
        low = every[every.float() <= top][-127 * 32:]
        low = torch.nn.functional.pad(low, (0, 127 * 32 - low.numel())).view(32, 127)
        lead = torch.full((32, 1), top).to(dtype)
        sign = torch.where(torch.arange(127) % 2 == 0, 1.0, -1.0).to(dtype)
        rows.append(torch.cat([lead, low * sign], 1).reshape(1, -1))
    tiny = every[:127 * 32].view(32, 127)   # subnormal numbers alone
    rows.append(torch.cat([every[127 * 32:127 * 32 + 32, None], tiny], 1).reshape(1, -1))
    x = torch.cat(rows)
    q, scale = ops.quantize_blocks(x.to(DEV))
    wq, ws = quantized(x)
    assert torch.equal(scale.cpu(), ws)
    assert same_codes(q, wq)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_zeros_infinities_and_nan(dtype):
    x = torch.zeros(6, 256)
    x[1, 5], x[1, 200] = float("inf"), -2.0
    x[2, 130], x[2, 131] = float("nan"), 1.0
    x[3, 0], x[3, 1] = float("-inf"), float("nan")
    x[4, 7] = 448.0
    x[5] = -0.0
    x = x.to(dtype)
    q, scale = ops.quantize_blocks(x.to(DEV))
    wq = torch.zeros(6, 256)
    wq[1, 5], wq[1, 200] = float("nan"), -448.0    # inf / inf; 0 beside an Inf is 0 / inf
    wq[2, 128:] = float("nan")
    wq[3, :128] = float("nan")
    wq[4, 7] = 448.0
    assert same_codes(q, wq)
    s = scale.cpu()
    assert s[0].tolist() == [1.0, 1.0] and s[4].tolist() == [1.0, 1.0] and s[5].tolist() == [1, 1]
    assert s[1, 0].item() == float("inf") and s[2, 0].item() == 1.0 and s[2, 1].isnan()
    assert s[3, 0].isnan() and s[3, 1].item() == 1.0


@pytest.mark.gpu
def test_quantize_strided_rows_and_no_rows():
    wide = torch.randn(20, 1024, generator=generator(3)).half().to(DEV)
    view = wide[::2, 64:64 + 272]
    q, scale = ops.quantize_blocks(view)
    wq, ws = quantized(view)
    assert same_codes(q, wq) and torch.equal(scale.cpu(), ws)
    q, scale = ops.quantize_blocks(wide[:0])
    assert q.shape == (0, 1024) and scale.shape == (0, 8)


# ----------------------------------------------------------------- gemm_blocks
def weights(N, K, seed):
    gen = generator(seed)
    W = (torch.randn(N, K, generator=gen) * 100).clamp_(-448, 448).to(FP8)
    return W, (torch.rand(blocks(N), blocks(K), generator=gen) + 0.5) * 0.01


def spread(scale, N, K):
    return scale.double().repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]


def reference(q, xs, W, ws):
    """(y, S) in 64 bits."""
    x = q.double() * xs.double().repeat_interleave(128, 1)[:, :q.shape[1]]
    w = W.double() * spread(ws, *W.shape)
    return x @ w.t(), x.abs() @ w.abs().t()


def near(y, want, S, K, cut=0.0):
    y = y.cpu()
    tol = HALF_STEP[y.dtype] * want.abs() + (K + 2) * 2.0 ** -23 * S + cut
    off = (y.double() - want).abs()
    assert (off <= tol).all(), f"{(off / tol).max()} of the tolerance at {(off / tol).argmax()}"


def instruction_cut(q, xs, W, ws):
    """What the matrix instruction's own sum may lose.  It adds eight products of
    consecutive k at a time, cut off (towards zero) 13 binary places below the leading
    one of the largest: seven of them lose less than 2^-13 of it each, the largest, a
    product of two numbers of 4 bits, nothing.  It is at most the largest |x| of the
    eight times the largest |w|.  (Over long rows the bound of the fp32 sums, which is
    K steps of all magnitudes together, is wider than this one.)"""
    x = q.double() * xs.double().repeat_interleave(128, 1)[:, :q.shape[1]]
    w = W.double() * spread(ws, *W.shape)
    x, w = (v.abs().view(v.shape[0], -1, 8).amax(2) for v in (x, w))
    return 7 * 2.0 ** -13 * (x @ w.t())


SIZES = [
    # T, N, K: one token to several tiles, short last blocks, odd outputs
    (1, 16, 16), (1, 130, 144), (1, 1, 128), (1, 4100, 4096), (2, 512, 640), (5, 77, 2064),
    (16, 256, 1024), (17, 129, 528), (33, 1000, 272), (48, 384, 4096), (64, 640, 1152),
    (65, 255, 512), (128, 128, 128), (129, 259, 400), (200, 1031, 2048), (257, 513, 1040),
    (300, 2048, 1536), (513, 700, 656), (1030, 1300, 784),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,N,K", SIZES)
def test_gemm_of_quantized_rows(dtype, T, N, K):
    W, ws = weights(N, K, N + K)
    q, xs = quantized(torch.randn(T, K, generator=generator(T)))
    # scales as quantize_blocks lays them out, and row by row
    y = ops.gemm_blocks(q.to(DEV), W.to(DEV), ws.to(DEV), x_scale=xs.t().contiguous().to(DEV).t(),
                        dtype=dtype)
    want, S = reference(q, xs, W, ws)
    assert y.dtype == dtype and y.shape == (T, N)
    near(y, want, S, K)
    again = ops.gemm_blocks(q.to(DEV), W.to(DEV), ws.to(DEV), x_scale=xs.to(DEV), dtype=dtype)
    assert torch.equal(y, again)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,N,K", SIZES)
def test_gemm_quantizes_on_the_way(dtype, T, N, K):
    W, ws = weights(N, K, N + K)
    x = (torch.randn(T, K, generator=generator(T)) * 2).to(dtype)
    y = ops.gemm_blocks(x.to(DEV), W.to(DEV), ws.to(DEV))
    want, S = reference(*quantized(x), W, ws)
    near(y, want, S, K)
    # the same as in two calls
    q, xs = ops.quantize_blocks(x.to(DEV))
    two = ops.gemm_blocks(q, W.to(DEV), ws.to(DEV), x_scale=xs, dtype=dtype)
    near(two, want, S, K)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,K", [(16, 4096), (16, 5120), (9, 8192), (4, 14336), (1, 16384),
                                 (16, 14336)])
def test_gemm_of_few_tokens_and_long_rows(dtype, T, K):
    """Rows that fill most of a CU's LDS, and those that do not fit it."""
    N = 200
    W, ws = weights(N, K, K)
    x = torch.randn(T, K, generator=generator(T)).to(dtype)
    q, xs = quantized(x)
    want, S = reference(q, xs, W, ws)
    near(ops.gemm_blocks(x.to(DEV), W.to(DEV), ws.to(DEV)), want, S, K)
    near(ops.gemm_blocks(q.to(DEV), W.to(DEV), ws.to(DEV), x_scale=xs.to(DEV), dtype=dtype), want,
         S, K)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,K", [(2, 16), (2, 128), (7, 112), (16, 16), (16, 128), (3, 144),
                                 (16, 256)])
def test_gemm_of_few_tokens_and_one_block(dtype, T, K):
    """Rows of one block, and of little more: a token's scales, whatever their strides."""
    N = 150
    W, ws = weights(N, K, K)
    x = torch.randn(T, K, generator=generator(T)).to(dtype)
    q, xs = quantized(x)
    want, S = reference(q, xs, W, ws)
    cut = instruction_cut(q, xs, W, ws)
    near(ops.gemm_blocks(x.to(DEV), W.to(DEV), ws.to(DEV)), want, S, K, cut)
    column = torch.full((T, 3 + blocks(K)), float("nan"))
    column[:, 3:] = xs
    for scale in (xs.to(DEV), xs.t().contiguous().to(DEV).t(), column.to(DEV)[:, 3:]):
        near(ops.gemm_blocks(q.to(DEV), W.to(DEV), ws.to(DEV), x_scale=scale, dtype=dtype), want,
             S, K, cut)


@pytest.fixture
def tuned():
    yield ops.tune
    ops.tune("blocks_shape", 0)
    ops.tune("blocks_parts", 0)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [1, 2, 3, 4])
@pytest.mark.parametrize("T,N,K", [(1, 16, 16), (5, 77, 2064), (33, 1000, 272), (200, 1031, 2048),
                                   (300, 2048, 1536), (513, 700, 656), (1100, 3000, 400)])
def test_gemm_of_every_tile_shape(tuned, shape, T, N, K):
    """Each shape of the tile kernel, whole rows and parts of them, also where another
    would be taken: tiles behind the ends, several tiles a workgroup, odd parts."""
    W, ws = weights(N, K, 3)
    q, xs = quantized(torch.randn(T, K, generator=generator(1)))
    want, S = reference(q, xs, W, ws)
    args = [t.to(DEV) for t in (q, W, ws)]
    tuned("blocks_shape", shape)
    for parts in (1, 2, 3, 5, 16):
        tuned("blocks_parts", parts)
        near(ops.gemm_blocks(*args, x_scale=xs.to(DEV)), want, S, K)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [5, 6, 7])
@pytest.mark.parametrize("T,N,K", [(1, 16, 16), (5, 77, 2064), (33, 1000, 272), (33, 30, 128),
                                   (200, 1031, 2048), (70, 2048, 1536), (513, 700, 656),
                                   (1100, 3000, 400), (20, 100, 144)])
def test_gemm_of_every_tile_shape_with_groups(tuned, shape, T, N, K):
    """The shapes whose waves have blocks of K in turn: blocks fewer than groups, odd
    ones, more workgroups than CUs; the groups add up in order."""
    W, ws = weights(N, K, 3)
    q, xs = quantized(torch.randn(T, K, generator=generator(1)))
    want, S = reference(q, xs, W, ws)
    cut = instruction_cut(q, xs, W, ws)
    args = [t.to(DEV) for t in (q, W, ws)]
    tuned("blocks_shape", shape)
    for parts in (1, 2, 3, 5, 16):
        tuned("blocks_parts", parts)
        y = ops.gemm_blocks(*args, x_scale=xs.to(DEV))
        near(y, want, S, K, cut)
        assert torch.equal(y, ops.gemm_blocks(*args, x_scale=xs.to(DEV)))


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [5, 6, 7])
def test_gemm_groups_without_a_block_add_nothing(tuned, shape):
    """The last block's scale is infinite, for one token and one block of outputs: the
    groups behind the end of K must not multiply it by zeros for anybody else."""
    T, N, K = 20, 160, 128 * 5
    W, ws = weights(N, K, 4)
    q, xs = quantized(torch.randn(T, K, generator=generator(1)))
    args = [t.to(DEV) for t in (q, W, ws)]
    tuned("blocks_shape", shape)
    clean = ops.gemm_blocks(*args, x_scale=xs.to(DEV)).cpu()
    xs[3, 4] = float("inf")
    got = ops.gemm_blocks(*args, x_scale=xs.to(DEV)).cpu()
    keep = [t for t in range(T) if t != 3]
    assert torch.equal(got[keep], clean[keep])
    # the sum of that block decides, whose sign is known
    part = (q[3, 512:].double() @ W[:, 512:].double().t())
    assert torch.equal(got[3], torch.where(part > 0, float("inf"), -float("inf")).half())


@pytest.mark.gpu
def test_gemm_of_more_tiles_than_workgroups(tuned):
    """A workgroup of 256 x 256 goes from one tile to the next: 300 of them."""
    T, N, K = 256 * 15 - 100, 256 * 20 - 60, 400
    W, ws = weights(N, K, 8)
    q, xs = quantized(torch.randn(T, K, generator=generator(2)))
    tuned("blocks_shape", 1)
    y = ops.gemm_blocks(q.to(DEV), W.to(DEV), ws.to(DEV), x_scale=xs.to(DEV))
    # some rows and columns of every tile
    rows, cols = torch.arange(0, T, 37), torch.arange(0, N, 41)
    want, S = reference(q[rows], xs[rows], W, ws)
    near(y.cpu()[rows][:, cols], want[:, cols], S[:, cols], K)
    tuned("blocks_shape", 0)
    near(ops.gemm_blocks(q.to(DEV), W.to(DEV), ws.to(DEV), x_scale=xs.to(DEV)).cpu()[rows], want,
         S, K)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 24, 300])
def test_gemm_rows_do_not_touch_each_other(T):
    """Inf, NaN and zeros of one token stay with it; those of a weight row with its output."""
    N, K = 260, 656
    W, ws = weights(N, K, 5)
    x = torch.randn(T, K, generator=generator(1)).half()
    clean = ops.gemm_blocks(x.to(DEV), W.to(DEV), ws.to(DEV)).cpu()
    bad = x.clone()
    bad[T // 2, 650] = float("nan")
    got = ops.gemm_blocks(bad.to(DEV), W.to(DEV), ws.to(DEV)).cpu()
    assert got[T // 2].isnan().all()
    keep = [t for t in range(T) if t != T // 2]
    assert torch.equal(got[keep], clean[keep])
    Wb = W.clone()
    Wb.view(torch.uint8)[255, 655] = 0x7F   # NaN in the last column
    got = ops.gemm_blocks(x.to(DEV), Wb.to(DEV), ws.to(DEV)).cpu()
    assert got[:, 255].isnan().all()
    assert torch.equal(got[:, :255], clean[:, :255]) and torch.equal(got[:, 256:], clean[:, 256:])
    zero = ops.gemm_blocks(torch.zeros_like(x).to(DEV), W.to(DEV), ws.to(DEV))
    assert (zero == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 7, 40, 600])
def test_gemm_strided_rows_out_and_one_row(T):
    N, K = 384, 512
    W, ws = (t.to(DEV) for t in weights(N, K, 9))
    wide = torch.randn(2 * T, K + 144, generator=generator(2)).bfloat16().to(DEV)
    x = wide[::2, 128:128 + K]
    plain = ops.gemm_blocks(x.contiguous(), W, ws)
    assert torch.equal(ops.gemm_blocks(x, W, ws), plain)
    guard = torch.full((T + 2, N), 7.0, dtype=torch.bfloat16, device=DEV)
    assert ops.gemm_blocks(x, W, ws, out=guard[1:T + 1]).data_ptr() == guard[1].data_ptr()
    assert torch.equal(guard[1:T + 1], plain) and (guard[0] == 7).all() and (guard[-1] == 7).all()
    q, xs = ops.quantize_blocks(x)
    wq = torch.zeros(2 * T, K + 64, dtype=torch.uint8, device=DEV).view(FP8)
    wq.view(torch.uint8)[::2, 16:16 + K] = q.view(torch.uint8)
    y = ops.gemm_blocks(wq[::2, 16:16 + K], W, ws, x_scale=xs, dtype=torch.bfloat16)
    assert torch.equal(y, ops.gemm_blocks(q, W.view(torch.uint8), ws, x_scale=xs,
                                          dtype=torch.bfloat16))
    one = ops.gemm_blocks(x[0], W, ws)
    assert one.shape == (N,) and torch.equal(one, ops.gemm_blocks(x[:1], W, ws)[0])
    assert ops.gemm_blocks(x[:0], W, ws).shape == (0, N)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 20, 200])
def test_gemm_in_a_graph_and_on_two_streams(T):
    N, K = 640, 2048
    W, ws = (t.to(DEV) for t in weights(N, K, 4))
    x = torch.randn(T, K, generator=generator(8)).half().to(DEV)
    ops.gemm_blocks(x, W, ws)
    g = torch.cuda.CUDAGraph()
    static = x.clone()
    with torch.cuda.graph(g):
        y = ops.gemm_blocks(static, W, ws)
    for seed in range(3):
        x = torch.randn(T, K, generator=generator(seed)).half().to(DEV)
        static.copy_(x)
        g.replay()
        assert torch.equal(y, ops.gemm_blocks(x, W, ws))
        torch.cuda.synchronize()
    xs = [torch.randn(T, K, generator=generator(20 + i)).half().to(DEV) for i in range(2)]
    want = [ops.gemm_blocks(v, W, ws) for v in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(ops.gemm_blocks(xs[i], W, ws))
    torch.cuda.synchronize()
    assert all(torch.equal(v, want[i]) for i in range(2) for v in got[i])


@pytest.mark.gpu
def test_quantized_weights_make_a_projection():
    """What quant gives for a matrix of a layer, through the product: within the two
    e4m3 roundings of a plain one."""
    gen = generator(6)
    Wf = torch.randn(1000, 1040, generator=gen) / 32
    x = torch.randn(40, 1040, generator=gen).half()
    W, ws = quant.quantize_e4m3_blocks(Wf.to(DEV))
    y = ops.gemm_blocks(x.to(DEV), W, ws).cpu().double()
    plain, S = x.double() @ Wf.double().t(), x.double().abs() @ Wf.double().abs().t()
    # a value is off by 2^-4 of itself, or 2^-10 scale where it is below 2^-6 scale
    # (at most 2^-10 / 448 of the block's largest); both factors, and the product of the two
    top_w = ws.cpu().double().repeat_interleave(128, 0)[:1000].repeat_interleave(128, 1)[:, :1040]
    top_x = quantized(x)[1].double().repeat_interleave(128, 1)[:, :1040]
    ew = Wf.double().abs() * 2.0 ** -4 + top_w * 2.0 ** -10
    ex = x.double().abs() * 2.0 ** -4 + top_x * 2.0 ** -10
    tol = x.double().abs() @ ew.t() + ex @ Wf.double().abs().t() + ex @ ew.t()
    assert ((y - plain).abs() <= tol + 2.0 ** -11 * y.abs() + 1042 * 2.0 ** -23 * S * 1.2).all()


def test_block_weights_on_the_cpu():
    W = torch.randn(2, 130, 272, generator=generator(1))
    W[0, :128, 128:256] = 0
    q, s = quant.quantize_e4m3_blocks(W)
    assert q.shape == W.shape and s.shape == (2, 2, 3) and s[0, 0, 1] == 1
    for e in range(2):
        for i in range(2):
            for j in range(3):
                part = W[e, 128 * i:128 * i + 128, 128 * j:128 * j + 128]
                if part.abs().max() > 0:
                    assert s[e, i, j] == part.abs().max() / 448
    back = quant.dequantize_e4m3_blocks(q, s)
    step = s.repeat_interleave(128, 1)[:, :130].repeat_interleave(128, 2)[..., :272]
    assert ((back - W).abs() <= W.abs() * (2.0 ** -4 + 2.0 ** -20) + step * 2.0 ** -10).all()
    with pytest.raises(ValueError):
        quant.quantize_e4m3_blocks(W[0, 0])


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_block_weights_that_are_not_finite_stay_visible(bad):
    """In their own block, whose numbers no scale holds beside them; no other changes."""
    W = torch.randn(256, 256, generator=generator(2)) / 50
    q0, s0 = quant.quantize_e4m3_blocks(W)
    W[3, 130] = bad
    q, s = quant.quantize_e4m3_blocks(W)
    back = quant.dequantize_e4m3_blocks(q, s)
    assert not s[0, 1].isfinite() and back[:128, 128:].isnan().all()
    s[0, 1] = s0[0, 1]
    assert torch.equal(s, s0)
    codes, codes0 = q.float(), q0.float()
    codes[:128, 128:] = codes0[:128, 128:] = 0
    assert torch.equal(codes, codes0)


# -------------------------------------------------------------------- refusals
P = 0x10000  # a fake, 256-byte aligned device address: never dereferenced


@pytest.fixture(scope="module")
def lib():
    from decodebench_amd import build

    if not ops.LIB_PATH.exists():
        build.build(verbose=False)
    return ops.load_library()


def test_quantize_contract(lib):
    def call(x=P, stride=256, q=P, scale=P, st=1, sb=4, T=4, K=256, dtype=0):
        return lib.db_quantize_blocks(x, stride, q, scale, st, sb, T, K, dtype, None)

    for bad in (dict(x=None), dict(q=None), dict(scale=None), dict(K=0), dict(K=24), dict(K=1 << 22),
                dict(stride=255), dict(stride=260), dict(stride=128), dict(T=-1), dict(T=1 << 22),
                dict(dtype=1), dict(dtype=7), dict(x=P + 2), dict(q=P + 8), dict(scale=P + 2),
                dict(st=-1), dict(st=0), dict(sb=0)):
        assert call(**bad) == ops.DB_ERR_INVALID, bad
        assert b"db_quantize_blocks" in lib.db_last_error()
    assert call(T=0, x=None, q=None, scale=None) == 0


def test_gemm_contract(lib):
    def call(x=P, stride=256, xs=P, st=1, sb=4, W=P, ws=P, y=P, T=4, K=256, N=64, xdt=1, ydt=0,
             work=None, nbytes=0):
        return lib.db_gemm_blocks(x, stride, xs, st, sb, W, ws, y, T, K, N, xdt, ydt, work, nbytes,
                                  None)

    for bad in (dict(x=None), dict(xs=None), dict(W=None), dict(ws=None), dict(y=None), dict(K=0),
                dict(K=40), dict(K=1 << 22), dict(N=0), dict(N=1 << 22), dict(T=-1),
                dict(T=1 << 22), dict(stride=240), dict(stride=264), dict(stride=1 << 23),
                dict(xdt=0), dict(xdt=2), dict(xdt=2, xs=None), dict(ydt=1), dict(ydt=9),
                dict(x=P + 8), dict(W=P + 8), dict(y=P + 4), dict(xs=P + 2), dict(ws=P + 1),
                dict(st=-1), dict(sb=-4), dict(st=1 << 22), dict(xdt=0, xs=None), dict(xdt=0, xs=None, work=P),
                dict(xdt=0, xs=None, work=P + 128, nbytes=1 << 20)):
        assert call(**bad) == ops.DB_ERR_INVALID, bad
        assert b"db_gemm_blocks" in lib.db_last_error()
    assert call(T=0, x=None, y=None, W=None, ws=None) == 0
    assert lib.db_gemm_blocks_workspace_bytes(0, 256, 64, 0) == 0


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 128, dtype=torch.float16)
    W, ws = torch.zeros(16, 128, dtype=FP8), torch.ones(1, 1)
    with pytest.raises((ValueError, RuntimeError)):
        ops.quantize_blocks(x)
    with pytest.raises((ValueError, RuntimeError)):
        ops.gemm_blocks(x, W, ws)
    with pytest.raises(TypeError):
        ops.quantize_blocks([1.0])
    with pytest.raises(TypeError):
        ops.gemm_blocks(None, W, ws)


@pytest.mark.gpu
def test_gemm_refusals():
    N, K, T = 64, 256, 4
    W, ws = (t.to(DEV) for t in weights(N, K, 1))
    x = torch.randn(T, K).half().to(DEV)
    q, xs = ops.quantize_blocks(x)
    for error, args, more in (
            (TypeError, (x.float(), W, ws), {}),
            (TypeError, (x, W.float(), ws), {}),
            (TypeError, (x, W, ws), dict(dtype=torch.bfloat16)),
            (TypeError, (q, W, ws), dict(x_scale=xs, dtype=torch.float32)),
            (ValueError, (q, W, ws), {}),
            (ValueError, (x, W, ws), dict(x_scale=xs)),
            (ValueError, (q, W, ws), dict(x_scale=xs[:, :1])),
            (ValueError, (q, W, ws), dict(x_scale=xs.double())),
            (ValueError, (q, W, ws), dict(x_scale=xs.cpu())),
            (ValueError, (x, W, None), {}),
            (ValueError, (x, W, ws[:, :1].contiguous()), {}),
            (TypeError, (x, W, ws.double()), {}),
            (ValueError, (x[:, :128], W, ws), {}),
            (ValueError, (x, W.t(), ws), {}),
            (ValueError, (x, W.view(torch.uint8)[:, ::2], ws), {}),
            (ValueError, (x[None], W, ws), {}),
            (ValueError, (x.t().contiguous().t(), W, ws), {}),
            (ValueError, (x[:, 4:132], W[:, :128].contiguous(), ws[:, :1].contiguous()), {}),
            (ValueError, (x, W, ws), dict(out=torch.empty(T, N + 1, dtype=x.dtype, device=DEV))),
            (TypeError, (x, W, ws), dict(out=torch.empty(T, N, device=DEV))),
            (ValueError, (x, W.cpu(), ws), {})):
        with pytest.raises(error):
            ops.gemm_blocks(*args, **more)
    with pytest.raises(TypeError):
        ops.quantize_blocks(x.float())
    with pytest.raises(ValueError):
        ops.quantize_blocks(x[:, :24])
    with pytest.raises(ValueError):
        ops.quantize_blocks(x[0])


def test_shared_memory_is_seen():
    """From the first element to the last, whatever the strides; neighbours are apart."""
    buf = torch.zeros(64, 32, dtype=torch.float16)
    out = buf[10:20]
    for other in (buf, out, buf[19:21], buf[::2], buf[0:11], buf[5:30, 8:16], out.view(torch.uint8)):
        with pytest.raises(ValueError, match="share memory with x"):
            ops._apart(out, (None, "none"), (other, "x"))
    ops._apart(buf[10:10], (buf, "around nothing"))
    ops._apart(out, (buf[:10], "before"), (buf[20:], "behind"), (buf[10:10], "nothing"),
               (buf.clone(), "another"), (buf[0:9:2], "rows before"))


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 8, 16, 40, 300])
def test_gemm_does_not_write_over_its_inputs(T):
    N = K = 256
    W, ws = (t.to(DEV) for t in weights(N, K, 1))
    buf = torch.randn(T + 8, K, generator=generator(2)).half().to(DEV)
    x, before = buf[4:T + 4], buf.clone()
    want = ops.gemm_blocks(x, W, ws)
    for out in (x, buf[3:T + 3], buf[5:T + 5])[:3 if T > 1 else 1]:
        with pytest.raises(ValueError, match="share memory"):
            ops.gemm_blocks(x, W, ws, out=out)
    with pytest.raises(ValueError, match="share memory"):   # one token from the middle of its row
        ops.gemm_blocks(x[0], W, ws, out=buf.view(-1)[4 * K + 8:5 * K + 8].view(1, N))
    q, xs = ops.quantize_blocks(x)
    codes = torch.empty(T * K * 2, dtype=torch.uint8, device=DEV)
    codes[:T * K] = q.view(torch.uint8).view(-1)
    with pytest.raises(ValueError, match="share memory"):
        ops.gemm_blocks(codes[:T * K].view(FP8).view(T, K), W, ws, x_scale=xs,
                        out=codes.view(torch.float16).view(T, N))
    assert torch.equal(buf, before)
    two = torch.empty(2 * T, N, dtype=torch.float16, device=DEV)
    two[:T] = x
    assert torch.equal(ops.gemm_blocks(two[:T], W, ws, out=two[T:]), want)


def test_the_oracle_sees_a_wrong_block():
    """The tolerance of a product is far below what one left-out block changes."""
    W, ws = weights(64, 512, 2)
    q, xs = quantized(torch.randn(4, 512, generator=generator(3)))
    want, S = reference(q, xs, W, ws)
    cut = q.clone()
    cut.view(torch.uint8)[:, 496:] = 0
    off, _ = reference(cut, xs, W, ws)
    tol = 2.0 ** -8 * want.abs() + 514 * 2.0 ** -23 * S
    assert ((off - want).abs() > tol).float().mean() > 0.9


def test_prototypes_take_their_arguments(lib):
    assert lib.db_gemm_blocks.argtypes[-2] is C.c_size_t


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 20, 100])
def test_native_call_path_and_python_steps_agree(T, monkeypatch):
    W, ws = (t.to(DEV) for t in weights(200, 528, 1))
    x = torch.randn(T, 528, generator=generator(5)).bfloat16().to(DEV)

    def calls():
        q, xs = ops.quantize_blocks(x)
        return (q.float(), xs, ops.gemm_blocks(x, W, ws), ops.gemm_blocks(q, W, ws, x_scale=xs),
                ops.gemm_blocks(q, W, ws, x_scale=xs, dtype=torch.bfloat16))

    ops.load_library()
    assert ops._fast is not None
    native = calls()
    monkeypatch.setattr(ops, "_fast", None)
    for a, b in zip(native, calls()):
        assert a.dtype == b.dtype and a.shape == b.shape and torch.equal(a, b)
        assert a.stride() == b.stride()
