"""Block-scaled 8-bit products and a mixture-of-experts layer: what they cost.

Every case is one call of a public entry point (``decodebench_amd.ops``):

* ``quant``  activations to OCP e4m3, one fp32 scale for each 128 elements of a
             row                                        (``ops.quantize_blocks``)
* ``gemm``   a projection on e4m3 weights with one fp32 scale for each block of
             128 x 128; activations of 16 bits, quantised on the way, or
             quantised already                          (``ops.gemm_blocks``)
* ``route``  the experts of each token and their weights    (``ops.moe_route``)
* ``moe``    a whole mixture-of-experts layer for a few tokens: router, gated
             experts, weighted sum                          (``ops.moe_layer``)

With ``own`` false, ``run`` computes the same in elementary torch operations.

Ranges: 1 to 8192 tokens of a projection, 1 to 512 of a layer; rows of 512 to
16384 elements (multiples of 16, so the last block of 128 may be short), 128 to
16384 outputs; 4 to 256 experts of 128 to 14336 channels, 1 to 8 for a token; fp16 and
bf16, experts of the same type or of block-scaled e4m3.
"""

import math

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
FP8 = torch.float8_e4m3fn
E4M3_MAX = 448.0
BLOCK = 128
# of a drawn case, about the largest listed one's
MOST_PRODUCTS = 8192 * 14336 * 4096
MOST_EXPERT_BYTES = 2_900_000_000
MOST_LAYER_FLOPS = 200_000_000_000


def _quant(name, dtype, T, K):
    return {"name": name, "op": "quant", "dtype": dtype, "T": T, "K": K}


def _gemm(name, dtype, x, T, N, K):
    return {"name": name, "op": "gemm", "dtype": dtype, "x": x, "T": T, "N": N, "K": K}


def _route(name, dtype, T, H, E, k, renormalize=True):
    return {"name": name, "op": "route", "dtype": dtype, "T": T, "H": H, "E": E, "k": k,
            "renormalize": renormalize}


def _moe(name, dtype, weights, T, H, I, E, k, renormalize=True):
    return {"name": name, "op": "moe", "dtype": dtype, "weights": weights, "T": T, "H": H,
            "I": I, "E": E, "k": k, "renormalize": renormalize}


def listed():
    return [
        # A decode step's activations of a few users: a call of pure latency.
        _quant("quant_t5", "f16", 5, 4096),
        # The activations of a long prompt before a down projection.
        _quant("quant_t8191", "bf16", 8191, 14336),
        # One user's token through an up projection: the bytes of the weights.
        _gemm("gemm_t1", "f16", "16bit", 1, 14336, 4096),
        # A serving batch through a fused qkv projection.
        _gemm("gemm_t48", "bf16", "16bit", 48, 6144, 4096),
        # Drafts and prompt pieces of several users, odd sizes, a down projection.
        _gemm("gemm_t301", "bf16", "fp8", 301, 4100, 14336),
        # A prompt's chunk; the largest: a long prompt through an up projection.
        _gemm("gemm_t2047", "f16", "16bit", 2047, 4096, 4096),
        _gemm("gemm_t8192", "bf16", "fp8", 8192, 14336, 4096),
        # One token among many experts; a batch of tokens, weights not renormalised.
        _route("route_t1", "bf16", 1, 4096, 128, 8),
        _route("route_t509", "f16", 509, 2048, 64, 6, renormalize=False),
        # One token through a layer of many small experts: latency and bytes.
        _moe("moe_t1", "bf16", "16bit", 1, 2048, 768, 128, 8),
        # A serving batch over many small experts of an odd width, quantised.
        _moe("moe_t33_fp8", "bf16", "fp8", 33, 2048, 1392, 64, 6),
        # The largest: a batch with prompt pieces through eight large experts.
        _moe("moe_t201", "f16", "16bit", 201, 4096, 14336, 8, 2),
    ]


def _log_int(rng, lo, hi, step=1):
    n = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return min(hi, max(lo, int(round(n / step)) * step))


def draw(rng):
    while True:
        op = rng.choice(("quant", "gemm", "gemm", "gemm", "route", "moe", "moe", "moe"))
        dtype = rng.choice(("f16", "bf16"))
        if op == "quant":
            case = {"op": op, "dtype": dtype, "T": _log_int(rng, 1, 8192),
                    "K": _log_int(rng, 512, 16384, 16)}
            return case
        if op == "gemm":
            case = {"op": op, "dtype": dtype, "x": rng.choice(("16bit", "fp8")),
                    "T": _log_int(rng, 1, 8192),
                    "N": _log_int(rng, 128, 16384, rng.choice((1, 4, 128))),
                    "K": _log_int(rng, 512, 16384, rng.choice((16, 128, 128)))}
            if case["T"] * case["N"] * case["K"] <= MOST_PRODUCTS:
                return case
            continue
        case = {"op": op, "dtype": dtype, "T": _log_int(rng, 1, 512),
                "H": _log_int(rng, 512, 8192, rng.choice((16, 128, 128))),
                "E": rng.choice((4, 8, 16, 32, 60, 64, 128, 128, 160, 256)),
                "renormalize": rng.choice((True, True, False))}
        case["k"] = rng.choice([k for k in (1, 2, 2, 4, 6, 8, 8) if k <= case["E"]])
        if op == "route":
            return case
        case |= {"weights": rng.choice(("16bit", "fp8")),
                 "I": _log_int(rng, 128, 14336, rng.choice((16, 128, 128)))}
        if (3 * case["E"] * case["I"] * case["H"] * (1 if case["weights"] == "fp8" else 2)
                <= MOST_EXPERT_BYTES and work(case)["flops"] <= MOST_LAYER_FLOPS):
            return case


def _blocks(n):
    return -(-n // BLOCK)


# ------------------------------------------------------------------- inputs
def _randn(gen, *shape, std=1.0, dtype=torch.float32):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32).mul_(std).to(dtype)


def _activations(gen, T, K, dtype):
    """Unit size, with some channels of far larger values, as a layer's
    activations have them."""
    x = _randn(gen, T, K)
    big = torch.rand(K, generator=gen, device="cuda") < 0.004
    return torch.where(big, x * 20.0, x).to(dtype)


def _block_weights(gen, *shape):
    """e4m3 weights [.., N, K] over most of the type's range and scales
    [.., N / 128, K / 128] that make them 1 / sqrt(K) in size."""
    N, K = shape[-2:]
    W = _randn(gen, *shape, std=100.0).clamp_(-E4M3_MAX, E4M3_MAX).to(FP8)
    s = torch.rand(*shape[:-2], _blocks(N), _blocks(K), generator=gen, device="cuda")
    return W, s.add_(0.5).mul_(0.01 / math.sqrt(K))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, T, dtype = case["op"], case["T"], DTYPES[case["dtype"]]
    if op == "quant":
        return {"op": op, "x": _activations(gen, T, case["K"], dtype)}
    if op == "gemm":
        W, ws = _block_weights(gen, case["N"], case["K"])
        x, xs = _activations(gen, T, case["K"], dtype), None
        if case["x"] == "fp8":
            # kept as quantize_blocks gives them: the scales of a block's tokens side by side
            x, xs = _quantized(x)
            xs = xs.t().contiguous().t()
        return {"op": op, "x": x, "xs": xs, "W": W, "ws": ws, "dtype": dtype}
    H, E = case["H"], case["E"]
    # Experts differ in how often they are asked: so do the sizes of the router's rows.
    size = torch.rand(E, 1, generator=gen, device="cuda").add_(0.5).div_(math.sqrt(H))
    s = {"op": op, "x": _randn(gen, T, H, dtype=dtype), "k": case["k"],
         "Wr": (_randn(gen, E, H) * size).to(dtype), "renormalize": case["renormalize"],
         "sg": None, "su": None, "sd": None}
    if op == "route":
        return s
    for w, sc, shape in (("Wg", "sg", (E, case["I"], H)), ("Wu", "su", (E, case["I"], H)),
                         ("Wd", "sd", (E, H, case["I"]))):
        if case["weights"] == "fp8":
            s[w], s[sc] = _block_weights(gen, *shape)
        else:
            s[w] = _randn(gen, *shape, std=1.0 / math.sqrt(shape[-1]), dtype=dtype)
    return s


# -------------------------------------------------------------- plain forms
def _quantized(x):
    T, K = x.shape
    f = x.float()
    wide = torch.nn.functional.pad(f, (0, _blocks(K) * BLOCK - K)).view(T, -1, BLOCK)
    scale = wide.abs().amax(-1) / E4M3_MAX
    scale = torch.where(scale == 0, torch.ones_like(scale), scale)
    q = (wide / scale[..., None]).clamp(-E4M3_MAX, E4M3_MAX).view(T, -1)[:, :K]
    return q.to(FP8), scale


def _spread(scale, N, K):
    """Block scales [.., N / 128, K / 128] for each weight [.., N, K]."""
    s = scale.repeat_interleave(BLOCK, -1)[..., :K]
    return s.repeat_interleave(BLOCK, -2)[..., :N, :]


def _gemm_plain(s):
    N, K = s["W"].shape
    x, xs = (s["x"], s["xs"]) if s["xs"] is not None else _quantized(s["x"])
    x = x.float() * xs.repeat_interleave(BLOCK, 1)[:, :K]
    return torch.matmul(x, (s["W"].float() * _spread(s["ws"], N, K)).t()).to(s["dtype"])


def _route_plain(s):
    # in 64 bits: the choice between two experts that are nearly alike
    logits = torch.matmul(s["x"].double(), s["Wr"].double().t())
    top, experts = torch.sort(logits, dim=-1, descending=True, stable=True)
    p = (top - top[:, :1]).float().exp()
    total = (p[:, :s["k"]] if s["renormalize"] else p).sum(-1, keepdim=True)
    return experts[:, :s["k"]].to(torch.int32), p[:, :s["k"]] / total


def _values(W, scale, experts):
    """The experts' weights in 32 bits."""
    if scale is None:
        return W[experts].float()
    w = W.view(torch.uint8)[experts].view(FP8).float()
    return w.mul_(_spread(scale[experts], *W.shape[1:]))


def _moe_plain(s):
    T, H = s["x"].shape
    E, k = s["Wr"].shape[0], s["k"]
    experts, weights = _route_plain(s)
    x, e = s["x"].float(), experts.flatten().long()
    if T * k <= E:
        # each token with its experts' weights
        which, rows = e, x.repeat_interleave(k, 0)[:, None]
        place = (torch.arange(T * k, device=x.device), torch.zeros_like(e))
    else:
        # each expert with its tokens, as a padded batch
        order = torch.argsort(e, stable=True)
        count = torch.bincount(e, minlength=E)
        at = torch.arange(T * k, device=x.device) - (torch.cumsum(count, 0) - count)[e[order]]
        rows = torch.zeros(E, int(count.max()), H, device=x.device)
        rows[e[order], at] = x[order // k]
        which, at = torch.arange(E, device=x.device), torch.empty_like(at).scatter_(0, order, at)
        place = (e, at)
    g = torch.bmm(rows, _values(s["Wg"], s["sg"], which).transpose(1, 2).contiguous())
    u = torch.bmm(rows, _values(s["Wu"], s["su"], which).transpose(1, 2).contiguous())
    h = g * torch.sigmoid(g) * u
    o = torch.bmm(h, _values(s["Wd"], s["sd"], which).transpose(1, 2).contiguous())[place]
    return (o.view(T, k, H) * weights[..., None]).sum(1).to(s["x"].dtype)


def run(state):
    s, op = state, state["op"]
    if own:
        from decodebench_amd import ops

        if op == "quant":
            q, scale = ops.quantize_blocks(s["x"])
            return {"q": q, "scale": scale}
        if op == "gemm":
            return ops.gemm_blocks(s["x"], s["W"], s["ws"], x_scale=s["xs"], dtype=s["dtype"])
        if op == "route":
            experts, weights = ops.moe_route(s["x"], s["Wr"], s["k"], renormalize=s["renormalize"])
            return {"experts": experts, "weights": weights}
        return ops.moe_layer(s["x"], s["Wr"], s["Wg"], s["Wu"], s["Wd"], s["k"],
                             renormalize=s["renormalize"], sg=s["sg"], su=s["su"], sd=s["sd"])
    if op == "quant":
        q, scale = _quantized(s["x"])
        return {"q": q, "scale": scale}
    if op == "gemm":
        return _gemm_plain(s)
    if op == "route":
        experts, weights = _route_plain(s)
        return {"experts": experts, "weights": weights}
    return _moe_plain(s)


# --------------------------------------------------------------------- work
def work(case):
    """Bytes: each input read once, each output written once; of the experts,
    as many as T tokens with k different ones each hit on average if all are
    equally likely.  Flops: two per multiply-add of the products."""
    op, T = case["op"], case["T"]
    if op == "quant":
        K = case["K"]
        return {"bytes": T * (2 * K + K + 4 * _blocks(K)), "flops": 2 * T * K}
    if op == "gemm":
        N, K = case["N"], case["K"]
        x = 2 * K if case["x"] == "16bit" else K + 4 * _blocks(K)
        return {"bytes": T * x + N * K + 4 * _blocks(N) * _blocks(K) + 2 * T * N,
                "flops": 2 * T * N * K}
    H, E, k = case["H"], case["E"], case["k"]
    route = {"bytes": 2 * T * H + 2 * E * H, "flops": 2 * T * E * H}
    if op == "route":
        return {"bytes": route["bytes"] + 8 * T * k, "flops": route["flops"]}
    I = case["I"]
    hit = E * (1.0 - (1.0 - k / E) ** T)
    one = 3 * H * I * 2 if case["weights"] == "16bit" else (
        3 * H * I + 12 * _blocks(H) * _blocks(I))
    return {"bytes": int(route["bytes"] + 2 * T * H + hit * one),
            "flops": route["flops"] + 6 * T * k * H * I}


# ------------------------------------------------------------ 64-bit results
def _quantized64(x):
    """Block after block, (codes' values, scales); the scale itself is defined
    in 32 bits."""
    q, scales = torch.empty_like(x, dtype=torch.float64), []
    for b in range(0, x.shape[1], BLOCK):
        part = x[:, b:b + BLOCK].double()
        s = (part.abs().max(dim=1).values.float() / E4M3_MAX).double()
        s[s == 0] = 1.0
        v = (part / s[:, None]).clamp(-E4M3_MAX, E4M3_MAX)
        # e4m3: three bits behind the leading one, steps of 2^-9 below 2^-6
        step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
        q[:, b:b + BLOCK] = torch.round(v / step) * step
        scales.append(s)
    return q, torch.stack(scales, 1)


def _weights64(W, scale):
    w = W.to(torch.float64)
    if scale is not None:
        for i in range(scale.shape[0]):
            for j in range(scale.shape[1]):
                w[i * BLOCK:(i + 1) * BLOCK, j * BLOCK:(j + 1) * BLOCK] *= scale[i, j].double()
    return w


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "quant":
        q, scale = _quantized64(s["x"])
        return {"q": q, "scale": scale}
    if op == "gemm":
        if s["xs"] is None:
            x, xs = _quantized64(s["x"])
        else:
            x, xs = s["x"].to(torch.float64), s["xs"].double()
        for b in range(xs.shape[1]):
            x[:, b * BLOCK:(b + 1) * BLOCK] *= xs[:, b:b + 1]
        return x @ _weights64(s["W"], s["ws"]).t()
    x, k, T = s["x"].double(), case["k"], case["T"]
    logits = x @ s["Wr"].double().t()
    p = torch.softmax(logits, -1)
    left, chosen, share = logits.clone(), [], []
    for _ in range(k):
        best = left.max(-1, keepdim=True).values
        at = (left == best).int().argmax(-1)
        chosen.append(at)
        share.append(p.gather(1, at[:, None])[:, 0])
        left.scatter_(1, at[:, None], -math.inf)
    chosen, share = torch.stack(chosen, 1), torch.stack(share, 1)
    if case["renormalize"]:
        share = share / share.sum(1, keepdim=True)
    if op == "route":
        return {"experts": chosen.to(torch.int32), "weights": share}
    y = torch.zeros(T, case["H"], dtype=torch.float64, device=x.device)
    for e in chosen.unique().tolist():
        t, j = torch.nonzero(chosen == e, as_tuple=True)
        Wg, Wu, Wd = (_weights64(s[w][e], None if s[sc] is None else s[sc][e])
                      for w, sc in (("Wg", "sg"), ("Wu", "su"), ("Wd", "sd")))
        g = x[t] @ Wg.t()
        h = g / (1 + torch.exp(-g)) * (x[t] @ Wu.t())
        y.index_add_(0, t, (h @ Wd.t()) * share[t, j][:, None])
    return y
