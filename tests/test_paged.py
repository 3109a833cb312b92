"""The operators of a serving step over a paged KV cache, against plain
implementations in 64 bits: ``paged_plan``, ``rope_append`` and
``paged_attention``, one by one, their refusals, and a step of all three.

Tolerances count roundings: u is half a step of the output's type (fp16 2^-11,
bf16 2^-8, e4m3 2^-4), relative to the value rounded.

* rope_append: one rounding of the result, and the fp32 sines, cosines and
  products, each within 2^-22 of |a| + |b| (u |y| + 2^-20 (|a| + |b|)).
* paged_attention: with A = sum_j p_j |v_j| / sum_j p_j, rounding the
  probabilities moves numerator and denominator by at most u A each, rounding
  the output by u |o| <= u A; fp32 sums and exponents of scores below 2^6 stay
  under 2^-13 A (3 u A + 2^-13 A).  What an e4m3 cache holds is exact in both.
"""

import ctypes as C
import math

import pytest

torch = pytest.importorskip("torch")

from decodebench_amd import ops  # noqa: E402

HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8,
             torch.float8_e4m3fn: 2.0 ** -4}
FP8 = torch.float8_e4m3fn
DEV = "cuda"


def ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=DEV)


# ------------------------------------------------------------------ paged_plan
def plan_reference(past, new, table, free, free_start, page, T):
    """The plan, one token after another."""
    R, width = len(past), len(table[0]) if table else 0
    table = [list(row) for row in table]
    position, slot, q_start, kv_len, taken, t = [], [], [0], [], free_start, 0
    for r in range(R):
        n = max(0, min(max(new[r], 0), T - t))
        old = max(past[r], 0)
        held = min(-(-old // page), width)
        for i in range(n):
            pos = old + i
            p = pos // page
            number = -1
            if p < width:
                if p >= held:
                    at = taken + p - held
                    number = free[at] if at < len(free) else -1
                    table[r][p] = number
                else:
                    number = table[r][p]
            position.append(pos)
            slot.append(number * page + pos % page if number >= 0 else -1)
        taken += min(-(-(old + n) // page), width) - held
        t += n
        q_start.append(t)
        kv_len.append(old + n)
    position += [0] * (T - t)
    slot += [-1] * (T - t)
    return q_start, kv_len, position, slot, taken, table


def check_plan(past, new, page, T, free, free_start=0, width=None, table=None, pad=0):
    R = len(past)
    if table is None:
        width = width or max(1, max((-(-(max(p, 0) + max(n, 0)) // page)
                                     for p, n in zip(past, new)), default=1))
        table = [[1000 + 100 * r + p if p < -(-max(past[r], 0) // page) else -7
                  for p in range(width)] for r in range(R)]
    want = plan_reference(past, new, table, free, free_start, page, T)
    wide = torch.full((R, width + pad), -9, dtype=torch.int32, device=DEV)
    view = wide[:, :width]
    if R:
        view.copy_(ints(table))
    got = ops.paged_plan(ints(past), ints(new), view, ints(free), page, T,
                         free_start=ints([free_start]) if free_start else None)
    for name, g, w in zip(("q_start", "kv_len", "position", "slot"), got, want):
        assert g.tolist() == w, name
    assert got.slot.dtype == torch.int64
    assert got.free_next.tolist() == [want[4]]
    assert view.tolist() == want[5]
    assert (wide[:, width:] == -9).all()
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("past,new,page", [
    ([0], [1], 16),
    ([15, 16, 17, 0, 31], [1, 1, 1, 1, 1], 16),
    ([5, 0, 300, 7], [0, 40, 3, 129], 16),
    ([0, 0, 0], [0, 0, 0], 16),
    ([3, 100, 64], [50, 1, 64], 24),
    ([9, 2], [5, 8], 1),
    ([0, 4096], [4097, 1], 128),
])
def test_plan_lays_out_tokens_and_pages(past, new, page):
    free = list(range(5000, 4000, -1))
    check_plan(past, new, page, sum(new), free)
    check_plan(past, new, page, sum(new) + 5, free, free_start=3, pad=3)   # rows behind the last


@pytest.mark.gpu
def test_plan_of_no_request_and_of_no_token():
    got = check_plan([], [], 16, 4, [1, 2], width=2)
    assert got.slot.tolist() == [-1] * 4
    check_plan([5, 9], [0, 0], 16, 0, [], width=2)


@pytest.mark.gpu
def test_plan_of_many_requests():
    """More requests than one round of the prefix sums holds, some of them long."""
    gen = torch.Generator().manual_seed(3)
    R = 2600
    past = torch.randint(0, 200, (R,), generator=gen).tolist()
    new = torch.randint(0, 4, (R,), generator=gen).tolist()
    new[1023], new[1024], new[2599] = 700, 0, 333
    free = torch.randperm(60000, generator=gen).to(torch.int32).tolist()
    check_plan(past, new, 16, sum(new) + 100, free, free_start=11)


@pytest.mark.gpu
def test_plan_without_room():
    """Pages run out, tables are too narrow, rows are too few, lengths negative."""
    check_plan([0, 0, 14], [40, 20, 4], 16, 64, [3, 4])            # two pages for six
    check_plan([0, 30], [100, 10], 16, 110, list(range(50)), width=3)
    check_plan([100], [5], 16, 5, [9], width=3, table=[[1, 2, 3]])    # longer than its row already
    check_plan([8, 8, 8], [10, 10, 10], 16, 17, list(range(50)))   # 17 rows for 30 tokens
    check_plan([-5, 6], [3, -2], 16, 8, list(range(9)))
    check_plan([0], [3], 16, 3, [])


@pytest.mark.gpu
def test_plan_keeps_entries_without_a_page():
    """A token in a page that the request should hold but does not gets no slot."""
    check_plan([5, 20], [2, 3], 16, 5, [8, 9], width=3, table=[[-1, -1, -1], [4, -1, -1]])


@pytest.mark.gpu
def test_a_plan_is_saved_and_loaded(monkeypatch):
    """A plan's tensors are saved together, and alone as what they hold, on the native
    call path as on the Python one."""
    import io

    table = ints([[7, -1, -1], [9, 8, -1]])
    args = (ints([3, 20]), ints([40, 2]), table, ints([4, 5, 6]), 16, 1000)

    def saved(what):
        out = io.BytesIO()
        torch.save(what, out)
        out.seek(0)
        return torch.load(out, weights_only=True), len(out.getvalue())

    ops.load_library()
    assert ops._fast is not None
    sizes = []
    for fast in (ops._fast, None):
        monkeypatch.setattr(ops, "_fast", fast)
        p = ops.paged_plan(*args)
        for got, w in zip(saved(tuple(p))[0], p):
            assert got.dtype == w.dtype and torch.equal(got, w)
        sizes.append(saved(p.kv_len)[1])
    assert sizes[0] == sizes[1]


@pytest.mark.gpu
def test_a_plan_of_lengths_in_memory_of_another_owner():
    """Inputs whose storage no allocator of torch's made."""
    args = [ints([3, 20]), ints([40, 2]), ints([[7, -1, -1], [9, 8, -1]]), ints([4, 5, 6])]
    want = ops.paged_plan(*args, 16, 50)
    args[2] = ints([[7, -1, -1], [9, 8, -1]])
    got = ops.paged_plan(*(torch.from_dlpack(x) for x in args), 16, 50)
    for g, w in zip(got, want):
        assert torch.equal(g, w)
    assert args[2].tolist() == [[7, 4, 5], [9, 8, -1]]


# ----------------------------------------------------------------- rope_append
def cache_pair(gen, pages, Hkv, page, D, dtype, layout="heads", dev=DEV):
    def one():
        shape = (pages, page, Hkv, D) if layout == "tokens" else (pages, Hkv, page, D)
        x = torch.randn(*shape, generator=gen) * (40.0 if dtype == FP8 else 1.0)
        x = x.to(dtype).to(dev)
        return x.permute(0, 2, 1, 3) if layout == "tokens" else x

    scales = (None, None)
    if dtype == FP8:
        scales = tuple((torch.rand(Hkv, generator=gen) * 0.03 + 0.01).to(dev) for _ in range(2))
    return one(), one(), *scales


def rope_reference(qkv, position, slot, K, V, freq, Hkv, axes, interleaved, ks, vs):
    """(q, K, V) in 64 bits and what their roundings act on: the magnitudes
    |a| + |b| of each turned element."""
    T, D, rot = qkv.shape[0], K.shape[3], 2 * freq.numel()
    x = qkv.double().cpu().view(T, -1, D)
    Hq = x.shape[1] - 2 * Hkv
    pos = position.double().cpu().view(-1, T)
    axis = torch.tensor(axes or [0] * (rot // 2))
    angle = pos[axis].t() * freq.double().cpu()
    co, si = angle.cos()[:, None], angle.sin()[:, None]
    y, mag = x.clone(), x.abs()
    first = slice(0, rot, 2) if interleaved else slice(0, rot // 2)
    second = slice(1, rot, 2) if interleaved else slice(rot // 2, rot)
    heads = slice(0, Hq + Hkv)
    a, b = x[:, heads, first], x[:, heads, second]
    y[:, heads, first], y[:, heads, second] = a * co - b * si, b * co + a * si
    mag[:, heads, first] = mag[:, heads, second] = a.abs() + b.abs()
    caches = []
    for cache, scale, h0 in ((K, ks, Hq), (V, vs, Hq + Hkv)):
        page = cache.shape[2]
        c, m = cache.to(torch.float64).cpu(), torch.zeros(cache.shape, dtype=torch.float64)
        if scale is not None:
            c = c * scale.double().cpu()[:, None, None]
        for t, s in enumerate(slot.tolist()):
            if 0 <= s < cache.shape[0] * page:
                rows = y[t, h0:h0 + Hkv].clone()
                if scale is not None:
                    most = 448.0 * scale.double().cpu()[:, None]
                    rows = torch.maximum(torch.minimum(rows, most), -most)
                c[s // page, :, s % page] = rows
                m[s // page, :, s % page] = mag[t, h0:h0 + Hkv]
        caches.append((c, m))
    return (y[:, :Hq], mag[:, :Hq]), *caches


def check_rope(T, Hq, Hkv, D, page, dtype, cache_dtype, rot=None, axes=None, n_axes=1,
               interleaved=False, layout="heads", strided=False, far=0, drop=(), seed=0, out=False):
    gen = torch.Generator().manual_seed(seed)
    rot = rot or D
    pages = T // page + 3
    K, V, ks, vs = cache_pair(gen, pages, Hkv, page, D, cache_dtype, layout)
    width = (Hq + 2 * Hkv) * D
    qkv = torch.randn(T, width + (24 if strided else 0), generator=gen).to(dtype).to(DEV)[:, :width]
    slot = torch.randperm(pages * page, generator=gen)[:T]
    for t, s in drop:
        slot[t] = s
    slot = slot.to(DEV)
    pos = torch.randint(0, 50, (n_axes, T), generator=gen).to(torch.int32) + far
    pos = pos.to(DEV) if n_axes > 1 else pos[0].to(DEV)
    freq = (10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)).float().to(DEV)
    want = rope_reference(qkv, pos, slot, K, V, freq, Hkv, axes, interleaved, ks, vs)
    before = K.clone(), V.clone()
    buf = torch.empty(T, Hq, D, dtype=dtype, device=DEV) if out else None
    q = ops.rope_append(qkv, pos, slot, K, V, freq, axes=axes, interleaved=interleaved, k_scale=ks,
                        v_scale=vs, out=buf)
    assert buf is None or q is buf
    assert q.dtype == dtype and q.shape == (T, Hq, D)
    tol = HALF_STEP[dtype] * want[0][0].abs() + 2.0 ** -20 * want[0][1] + 2.0 ** -25
    assert ((q.double().cpu() - want[0][0]).abs() <= tol).all()
    for cache, old, scale, (w, mag) in ((K, before[0], ks, want[1]), (V, before[1], vs, want[2])):
        got = cache.to(torch.float64).cpu()
        floor = 2.0 ** -25
        if scale is not None:
            got = got * scale.double().cpu()[:, None, None]
            # half a step of the smallest e4m3 numbers, and the fp32 quotient
            floor = 2.0 ** -10 * scale.double().cpu()[:, None, None]
        tol = HALF_STEP[cache.dtype] * w.abs() + 2.0 ** -20 * mag + floor
        assert ((got - w).abs() <= tol).all()
        kept = (mag == 0).all(-1).to(DEV)          # rows that no token names
        assert torch.equal(cache.view(torch.uint8)[kept] if cache.dtype == FP8 else cache[kept],
                           old.view(torch.uint8)[kept] if cache.dtype == FP8 else old[kept])
    return q, K, V


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("T,Hq,Hkv,D,page", [
    (1, 32, 8, 128, 16), (3, 4, 4, 64, 1), (37, 10, 2, 128, 24), (1200, 5, 1, 64, 16),
    (5, 3, 3, 80, 7), (2, 2, 1, 256, 16), (9, 4, 2, 16, 5)])
def test_rope_append(dtype, fp8, T, Hq, Hkv, D, page):
    check_rope(T, Hq, Hkv, D, page, dtype, FP8 if fp8 else dtype)
    check_rope(T, Hq, Hkv, D, page, dtype, FP8 if fp8 else dtype, interleaved=True,
               layout="tokens", strided=True, seed=1, out=True)


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rot,axes,n_axes", [
    (64, None, 1), (16, None, 1), (128, [0] * 16 + [1] * 24 + [2] * 24, 3),
    (128, [i % 3 for i in range(64)], 3), (96, [3, 1] * 24, 4), (32, [0] * 16, 2)])
def test_rope_append_parts_and_axes(interleaved, rot, axes, n_axes):
    check_rope(21, 4, 2, 128, 16, torch.float16, torch.float16, rot=rot, axes=axes, n_axes=n_axes,
               interleaved=interleaved)


@pytest.mark.gpu
@pytest.mark.parametrize("far", [-40, 100_000, 2 ** 30])
def test_rope_append_far_positions(far):
    check_rope(17, 4, 2, 64, 16, torch.float16, torch.float16, far=far)


@pytest.mark.gpu
def test_rope_append_without_a_slot():
    """Slots outside the cache write nothing, their queries are turned all the same."""
    check_rope(20, 4, 2, 128, 16, torch.bfloat16, torch.bfloat16,
               drop=((0, -1), (7, 64), (8, 2 ** 40), (19, -2 ** 40)))


@pytest.mark.gpu
def test_rope_append_e4m3_saturates_and_keeps_nan():
    gen = torch.Generator().manual_seed(0)
    K, V, ks, vs = cache_pair(gen, 2, 1, 16, 64, FP8)
    qkv = torch.zeros(1, 3 * 64, dtype=torch.float16, device=DEV)
    qkv[0, 128:132] = torch.tensor([60000.0, -60000.0, math.nan, math.inf], device=DEV)
    freq = torch.ones(32, device=DEV)
    ops.rope_append(qkv, ints([3]), ints([17], torch.int64), K, V, freq, k_scale=ks, v_scale=vs)
    row = V[1, 0, 1].float().tolist()
    assert row[:2] == [448.0, -448.0] and math.isnan(row[2]) and row[3] == 448.0
    assert row[4:] == [0.0] * 60


@pytest.mark.gpu
def test_rope_append_of_no_token():
    gen = torch.Generator().manual_seed(0)
    K, V, *_ = cache_pair(gen, 2, 2, 16, 64, torch.float16)
    q = ops.rope_append(torch.empty(0, 6 * 64, dtype=torch.float16, device=DEV), ints([]),
                        ints([], torch.int64), K, V, torch.ones(32, device=DEV))
    assert q.shape == (0, 2, 64)


# ------------------------------------------------------------- paged_attention
def attention_reference(q, K, V, table, q_start, kv_len, scale, causal, window, ks, vs):
    """(o, A) in 64 bits, request by request; rows of no request are None (NaN)."""
    T, Hq, D = q.shape
    pages, Hkv, page, _ = K.shape
    G = Hq // Hkv
    q = q.double().cpu()
    o = torch.full((T, Hq, D), math.nan, dtype=torch.float64)
    size = torch.zeros(T, Hq, D, dtype=torch.float64)
    table, q_start, kv_len = table.cpu(), q_start.tolist(), kv_len.tolist()
    for r, L in enumerate(kv_len):
        lo, hi = q_start[r], q_start[r + 1]
        n, L = hi - lo, max(L, 0)
        j = torch.arange(min(L, table.shape[1] * page))
        number = table[r, j // page].long()
        there = (number >= 0) & (number < pages)
        j, number = j[there], number[there].to(K.device)
        off = (j % page).to(K.device)
        k = K.view(torch.uint8)[number, :, off].view(FP8) if K.dtype == FP8 else K[number, :, off]
        v = V.view(torch.uint8)[number, :, off].view(FP8) if V.dtype == FP8 else V[number, :, off]
        k, v = k.to(torch.float64).cpu(), v.to(torch.float64).cpu()
        if ks is not None:
            k = k * ks.double().cpu()[:, None]
            v = v * vs.double().cpu()[:, None]
        for i in range(n):
            pos = L - n + i
            seen = (j <= pos) if causal else torch.ones_like(j, dtype=torch.bool)
            if window:
                seen &= j > pos - window
            if not seen.any():
                o[lo + i] = 0.0
                continue
            ki, vi = k[seen], v[seen]
            for h in range(Hkv):
                s = q[lo + i, h * G:(h + 1) * G] @ ki[:, h].t() * scale
                p = torch.softmax(s, -1)
                o[lo + i, h * G:(h + 1) * G] = p @ vi[:, h]
                size[lo + i, h * G:(h + 1) * G] = p @ vi[:, h].abs()
    return o, size


def make_step(requests, Hq, Hkv, D, page, dtype, cache_dtype, layout="heads", seed=0, spare=3,
              std=1.0, extra=0):
    """Inputs of a call: requests [(new, length)], pages in random order; free
    pages and the places behind a length hold NaN."""
    gen = torch.Generator().manual_seed(seed)
    held = [-(-L // page) for _, L in requests]
    pages = sum(held) + spare
    K, V, ks, vs = cache_pair(gen, pages, Hkv, page, D, cache_dtype, layout)
    order = torch.randperm(pages, generator=gen).tolist()
    width = max(max(held, default=1), 1) + 1
    table, at = [], 0
    used = torch.zeros(pages, page, dtype=torch.bool)
    for (_, L), n in zip(requests, held):
        mine = order[at:at + n]
        at += n
        table.append(mine + [-1] * (width - n))
        for p, number in enumerate(mine):
            used[number, :max(0, min(page, L - p * page))] = True
    for cache in (K, V):
        c = cache.view(torch.uint8) if cache_dtype == FP8 else cache
        hide = (~used).to(DEV)[:, None, :, None].expand(cache.shape)
        c.masked_fill_(hide, 0x7F if cache_dtype == FP8 else math.nan)
    starts = [0]
    for n, _ in requests:
        starts.append(starts[-1] + n)
    q = (torch.randn(starts[-1] + extra, Hq, D, generator=gen) * std).to(dtype).to(DEV)
    return dict(q=q, K=K, V=V, block_table=ints(table), q_start=ints(starts),
                kv_len=ints([L for _, L in requests]), k_scale=ks, v_scale=vs)


def check_attention(s, causal=True, window=None, scale=None, want=None, **kw):
    q = s["q"]
    if want is None:
        want = attention_reference(q, s["K"], s["V"], s["block_table"], s["q_start"], s["kv_len"],
                                   1.0 / math.sqrt(q.shape[2]) if scale is None else scale, causal,
                                   window, s["k_scale"], s["v_scale"])
    o, size = want
    got = ops.paged_attention(**s, causal=causal, window=window, scale=scale, **kw)
    assert got.dtype == q.dtype and got.shape == q.shape
    g = got.double().cpu()
    rows = ~torch.isnan(o).all(-1).all(-1)          # rows of some request
    u = HALF_STEP[q.dtype]
    tol = (3 * u + 2.0 ** -13) * size + 2.0 ** -24
    bad = ~((g - o).abs() <= tol) & rows[:, None, None] & ~torch.isnan(o)
    assert not bad.any(), (bad.nonzero()[:4].tolist(),
                           ((g - o).abs() / tol)[bad][:4].tolist())
    return got


SINGLES = [(1, 1), (1, 15), (1, 16), (1, 17), (1, 200), (1, 64), (1, 333)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("Hq,Hkv,D,page", [
    (32, 8, 128, 16), (4, 4, 64, 32), (10, 2, 128, 24), (16, 1, 64, 1), (40, 2, 128, 128)])
def test_attention_of_single_tokens(dtype, fp8, Hq, Hkv, D, page):
    s = make_step(SINGLES, Hq, Hkv, D, page, dtype, FP8 if fp8 else dtype)
    check_attention(s)
    check_attention(s, max_new=1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("Hq,Hkv,D,page", [
    (8, 2, 128, 16), (3, 3, 64, 24), (5, 1, 128, 100), (16, 2, 64, 8)])
def test_attention_of_chunks(dtype, fp8, Hq, Hkv, D, page):
    requests = [(70, 70), (1, 90), (0, 50), (33, 290), (5, 5), (129, 140), (2, 64)]
    s = make_step(requests, Hq, Hkv, D, page, dtype, FP8 if fp8 else dtype, layout="tokens")
    want = attention_reference(s["q"], s["K"], s["V"], s["block_table"], s["q_start"],
                               s["kv_len"], 1.0 / math.sqrt(D), True, None, s["k_scale"],
                               s["v_scale"])
    check_attention(s, want=want)
    check_attention(s, want=want, max_new=129)
    check_attention(s, want=want, max_new=1)          # a broken promise costs only time


@pytest.mark.gpu
@pytest.mark.parametrize("n,L", [(1, 1), (2, 2), (4, 1000), (128, 128), (200, 1500), (1, 5000)])
def test_attention_of_one_request(n, L):
    """One request alone: its keys are split over workgroups."""
    check_attention(make_step([(n, L)], 8, 2, 128, 16, torch.float16, torch.float16, std=2.0))


@pytest.mark.gpu
@pytest.mark.parametrize("window", [1, 2, 16, 63, 64, 65, 100, 5000])
@pytest.mark.parametrize("D", [64, 128])
def test_attention_windows(window, D):
    requests = [(1, 300), (40, 200), (3, 77), (1, 5), (100, 100)]
    s = make_step(requests, 4, 2, D, 16, torch.float16, torch.float16)
    check_attention(s, window=window)
    check_attention(make_step([(1, 900), (1, 1), (3, 450)], 4, 2, D, 24, torch.float16,
                              torch.float16), window=window, max_new=3)


@pytest.mark.gpu
def test_attention_without_causal():
    requests = [(30, 100), (1, 50), (64, 64), (4, 4)]
    check_attention(make_step(requests, 8, 2, 128, 16, torch.bfloat16, torch.bfloat16),
                    causal=False, scale=0.3)


@pytest.mark.gpu
@pytest.mark.parametrize("max_new", [None, 1])
def test_attention_rows_that_see_nothing_and_rows_of_nobody(max_new):
    """Empty requests, more new tokens than length, padded requests, rows behind
    the last one."""
    s = make_step([(1, 40), (1, 30), (2, 20), (30, 60)], 4, 2, 64, 16, torch.float16,
                  torch.float16, extra=6)
    s["kv_len"] = ints([40, 0, 1, 20])               # none, one token too few, ten too few
    s["out"] = torch.full_like(s["q"], 7.0)
    got = check_attention(s, max_new=max_new)
    assert (got[1] == 0).all() and (got[2] == 0).all() and (got[4:14] == 0).all()
    assert (got[34:] == 7.0).all()
    s["kv_len"] = ints([-3, 0, -1, 0])
    got = ops.paged_attention(**s, max_new=max_new)
    assert (got[:34] == 0).all() and (got[34:] == 7.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("max_new", [None, 1])
@pytest.mark.parametrize("page", [16, 24, 128])
def test_attention_of_missing_pages(page, max_new):
    """Pages that are not in the cache are not seen, whatever their number."""
    s = make_step([(1, 400), (1, 300), (20, 390), (1, 100)], 4, 2, 128, page, torch.float16,
                  torch.float16)
    t = s["block_table"]
    t[0, 1], t[0, 0], t[1, 1], t[2, 0] = -1, 10 ** 9, -2 ** 31, s["K"].shape[0]
    t[3] = -1
    check_attention(s, max_new=max_new)
    # lengths that the table's row cannot hold
    s["kv_len"] = ints([400, 10 ** 6, 390, 2 ** 31 - 1])
    check_attention(s, max_new=max_new)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, FP8])
@pytest.mark.parametrize("n", [3, 40])
def test_attention_hidden_inf_and_nan(dtype, n):
    """Inf and NaN in the keys and values of tokens that a row does not see do
    not reach it; the rows that do see them show them."""
    act = torch.float16 if dtype == FP8 else dtype
    s = make_step([(n, 100), (1, 50)], 4, 2, 64, 16, act, dtype)
    want = attention_reference(s["q"], s["K"], s["V"], s["block_table"], s["q_start"],
                               s["kv_len"], 0.125, True, None, s["k_scale"], s["v_scale"])

    def put(cache, r, j, h, d, value):
        page = int(s["block_table"][r, j // 16])
        if cache.dtype == FP8:
            cache.view(torch.uint8)[page, h, j % 16, d] = 0x7F
        else:
            cache[page, h, j % 16, d] = value

    last = 99
    put(s["V"], 0, last, 0, 5, math.inf)
    put(s["V"], 0, last - 1, 1, 6, math.nan)
    put(s["K"], 0, last, 1, 7, math.nan)
    got = ops.paged_attention(**s).double().cpu()
    o, size = want
    o[n - 1, 0:2, 5] = math.nan if dtype == FP8 else math.inf
    o[n - 2:n, 2:4, 6] = math.nan
    o[n - 1, 2:4] = math.nan
    fine = torch.isfinite(o)
    tol = (3 * HALF_STEP[act] + 2.0 ** -13) * size + 2.0 ** -24
    assert ((got - o).abs() <= tol)[fine].all()
    assert torch.equal(got[~fine].isnan(), o[~fine].isnan())
    assert torch.equal(got[~fine].isinf(), o[~fine].isinf())


@pytest.mark.gpu
def test_attention_window_hides_inf_and_nan_before_it():
    s = make_step([(1, 300), (20, 200)], 4, 2, 64, 16, torch.float16, torch.float16)
    want = attention_reference(s["q"], s["K"], s["V"], s["block_table"], s["q_start"],
                               s["kv_len"], 0.125, True, 50, None, None)
    for r, upto in ((0, 250), (1, 131)):       # keys that no row of the request sees
        for j in range(upto):
            page = int(s["block_table"][r, j // 16])
            s["K"][page, :, j % 16] = math.nan
            s["V"][page, :, j % 16] = math.inf
    check_attention(s, window=50, want=want)


@pytest.mark.gpu
def test_attention_strides():
    """q inside a projection's rows, K and V inside one allocation, a table with
    a row stride, one row of the table for two requests."""
    s = make_step([(3, 60), (3, 60)], 4, 2, 64, 16, torch.float16, torch.float16, std=1.5)
    qkv = torch.randn(6, 8, 64, device=DEV).half()
    qkv[:, :4] = s["q"]
    both = torch.stack([s["K"], s["V"]], 1)
    s["q"], s["K"], s["V"] = qkv[:, :4], both[:, 0], both[:, 1]
    s["block_table"] = torch.cat([s["block_table"], s["block_table"]], 1)[:, :5]
    check_attention(s)
    s["q"] = qkv.transpose(0, 1).contiguous().transpose(0, 1)[:, :4]
    s["block_table"] = s["block_table"][:1].expand(2, 5)
    check_attention(s)


@pytest.mark.gpu
def test_attention_of_many_requests():
    """More requests than one round of the work search holds; a few long ones."""
    gen = torch.Generator().manual_seed(5)
    lens = torch.randint(1, 60, (700,), generator=gen).tolist()
    lens[3], lens[300], lens[699] = 3000, 2100, 900
    requests = [(1 if r % 9 else 0, L) for r, L in enumerate(lens)]
    requests[511], requests[10] = (37, 60), (20, 20)
    s = make_step(requests, 4, 2, 64, 16, torch.float16, torch.float16)
    check_attention(s)
    check_attention(s, max_new=37)


@pytest.mark.gpu
@pytest.mark.parametrize("D,L", [(64, 5000), (128, 4300)])
def test_attention_of_long_splits(D, L):
    """So many heads that a wave walks more tiles than its lanes hold places for."""
    requests = [(1, L - 13 * r) for r in range(20)]
    check_attention(make_step(requests, 32, 32, D, 16, torch.float16, torch.float16), max_new=1)


@pytest.mark.gpu
def test_attention_offsets_past_32_bits():
    """Pages behind 2^31 elements (and 2^32 bytes) of a long cache."""
    Hkv, page, D = 8, 64, 128
    pages = 2 ** 31 // (Hkv * page * D) + 40
    K = torch.empty(pages, Hkv, page, D, dtype=torch.float16, device=DEV)
    V = torch.empty_like(K)
    gen = torch.Generator().manual_seed(1)
    small = make_step([(1, 200), (40, 130)], 16, Hkv, D, page, torch.float16, torch.float16)
    n = small["K"].shape[0]
    far = pages - n
    K[far:], V[far:] = small["K"], small["V"]
    t = small["block_table"]
    want = attention_reference(small["q"], small["K"], small["V"], t, small["q_start"],
                               small["kv_len"], 1 / math.sqrt(D), True, None, None, None)
    s = dict(small, K=K, V=V, block_table=torch.where(t >= 0, t + far, t))
    check_attention(s, want=want)
    qkv = torch.randn(2, 32 * D, generator=gen).half().to(DEV)
    slot = ints([pages * page - 1, (pages - 2) * page], torch.int64)
    ops.rope_append(qkv, ints([0, 0]), slot, K, V, torch.ones(64, device=DEV))
    assert torch.equal(V[-1, :, -1], qkv.view(2, 32, D)[0, 24:])
    assert torch.equal(K[-2, :, 0], qkv.view(2, 32, D)[1, 16:24])


@pytest.mark.gpu
def test_attention_of_nothing():
    s = make_step([(1, 5)], 4, 2, 64, 16, torch.float16, torch.float16)
    s["q"] = s["q"][:0]
    s["q_start"] = ints([0, 0])
    assert ops.paged_attention(**s).shape == (0, 4, 64)
    s = make_step([(1, 5)], 4, 2, 64, 16, torch.float16, torch.float16)
    s.update(block_table=s["block_table"][:0], q_start=ints([0]), kv_len=ints([]),
             out=torch.full_like(s["q"], 3.0))
    assert (ops.paged_attention(**s) == 3.0).all()


@pytest.mark.gpu
def test_attention_is_the_same_every_time():
    s = make_step([(1, 3000), (60, 700), (1, 20)], 8, 2, 128, 16, torch.float16, torch.float16)
    first = ops.paged_attention(**s)
    for _ in range(5):
        assert torch.equal(ops.paged_attention(**s), first)


DRAFTS = [(20, 20), (12, 300), (5, 37), (1, 64), (0, 9), (20, 333), (11, 4)]


@pytest.mark.gpu
@pytest.mark.parametrize("window", [None, 1, 31, 33, 100])
@pytest.mark.parametrize("Hq,Hkv,D,page,dtype,cache", [
    (6, 2, 128, 16, torch.float16, torch.float16), (3, 1, 64, 24, torch.bfloat16, torch.bfloat16),
    (6, 2, 64, 32, torch.bfloat16, FP8), (3, 1, 128, 20, torch.float16, FP8)])
def test_attention_of_drafts(window, Hq, Hkv, D, page, dtype, cache):
    """Up to 60 rows a request: the keys of a tile are shared by two waves, and of
    some tiles one of the two sees nothing."""
    s = make_step(DRAFTS, Hq, Hkv, D, page, dtype, cache)
    check_attention(s, window=window, max_new=20)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, FP8])
def test_attention_of_drafts_hidden_inf_and_nan(dtype):
    test_attention_hidden_inf_and_nan(dtype, 20)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 5, 40])
@pytest.mark.parametrize("page", [16, 24])
def test_attention_of_the_longest_window(n, page):
    """A window of 2^31 - 1 hides nothing, also where a request has more new
    tokens than its length, so that the first of them lie before its start."""
    s = make_step([(n, 90), (n, 60)], 4, 2, 64, page, torch.float16, torch.float16)
    s["kv_len"] = ints([max(1, n - 3), 60])
    for window in (2 ** 31 - 1, 2 ** 31 - 2, 2 ** 40):
        check_attention(s, window=window, want=attention_reference(
            s["q"], s["K"], s["V"], s["block_table"], s["q_start"], s["kv_len"], 1 / 8.0, True, None,
            None, None), max_new=n)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,D", [(torch.float16, 128), (torch.bfloat16, 64)])
@pytest.mark.parametrize("n,L", [
    # rows of 3 heads over one KV head: a tile of 64, or one and a bit of 256; 4 to
    # over 100 tiles of 64 keys
    (20, 300), (20, 700), (20, 1100), (20, 2600), (20, 7000), (90, 500), (90, 1000), (90, 2200),
    (90, 4000), (90, 7000)])
def test_attention_of_split_chunks(n, L, dtype, D):
    """Rows joined from 1 to over 16 splits, some of which see nothing."""
    s = make_step([(n, L)], 3, 1, D, 16, dtype, dtype)
    check_attention(s)
    check_attention(s, window=400)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 30, 500])
def test_attention_of_one_request_and_many_rows_of_nobody(n):
    """Rows enough to fill the chip, most of them behind the request's last."""
    s = make_step([(n, 3000)], 8, 8, 64, 16, torch.float16, torch.float16, extra=9000 - n)
    s["out"] = torch.full_like(s["q"], 7.0)
    got = check_attention(s)
    assert (got[n:] == 7.0).all()


@pytest.mark.gpu
def test_attention_of_other_heads_in_a_workspace_as_large():
    """Calls whose workspaces have one size and tickets of different numbers."""
    few = make_step([(1, 3000), (1, 2500)], 17, 17, 128, 16, torch.float16, torch.float16)
    many = make_step([(1, 200 + 9 * r) for r in range(8)], 33, 33, 64, 16, torch.float16,
                     torch.float16)
    a, b = ops.paged_attention(**few, max_new=1), ops.paged_attention(**many, max_new=1)
    for _ in range(3):
        assert torch.equal(check_attention(few, max_new=1), a)
        assert torch.equal(check_attention(many, max_new=1), b)


@pytest.mark.gpu
@pytest.mark.parametrize("max_new", [None, 1])
def test_attention_of_rows_in_no_order(max_new):
    """A q_start that goes back or past the rows: requests without rows, and the
    others' rows as they should be."""
    s = make_step([(4, 50), (0, 40), (5, 60), (1, 20)], 4, 2, 64, 16, torch.float16, torch.float16)
    want = attention_reference(s["q"], s["K"], s["V"], s["block_table"], s["q_start"],
                               s["kv_len"], 1 / 8.0, True, None, None, None)
    s["out"] = torch.full_like(s["q"], 7.0)
    s["q_start"] = ints([0, 4, -9, 2 ** 31 - 1, -2 ** 31])
    assert ops.paged_attention(**s, max_new=max_new).isfinite().all()
    s["q_start"] = ints([-5, 4, 4, 9, 2 ** 31 - 1])      # the same rows once clamped
    check_attention(s, want=want, max_new=max_new)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,cache,D,page", [
    (torch.float16, torch.float16, 128, 16), (torch.bfloat16, torch.bfloat16, 64, 24),
    (torch.bfloat16, FP8, 128, 32)])
def test_attention_of_prompts_from_nothing(dtype, cache, D, page):
    """No past: the row tiles of a request see anything from one tile of keys to all."""
    check_attention(make_step([(900, 900)], 8, 2, D, page, dtype, cache))
    check_attention(make_step([(330, 330), (1, 1), (515, 515), (64, 64)], 8, 2, D, page, dtype,
                              cache), max_new=515)


@pytest.mark.gpu
@pytest.mark.parametrize("max_new", [None, 1, 3])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("G", [7, 64, 300])
def test_attention_of_many_heads_over_one(G, D, max_new):
    """A token's rows fill a row tile, or several."""
    s = make_step([(1, 200), (3, 90), (2, 33), (0, 4)], G, 1, D, 16, torch.bfloat16, FP8)
    check_attention(s, max_new=max_new)


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("max_new", [None, 1, 8])
def test_attention_of_a_row_of_q_that_is_not_finite(bad, max_new):
    """It shows in its own row and head and nowhere else."""
    for requests in ([(1, 300), (1, 40), (1, 700)], [(20, 300), (1, 40), (30, 70)],
                     [(2, 300), (3, 40)]):
        s = make_step(requests, 8, 2, 64, 16, torch.float16, torch.float16)
        o, size = attention_reference(s["q"], s["K"], s["V"], s["block_table"], s["q_start"],
                                      s["kv_len"], 1 / 8.0, True, None, None, None)
        s["q"][-1, 3] = bad
        o[-1, 3] = math.nan
        got = check_attention(s, want=(o, size), max_new=max_new)
        assert got[-1, 3].isnan().all()


# ------------------------------------------------------- rows counted twice
# How paged_attention sizes a call from T and R alone, and what its kernels then
# find in q_start: a model on the CPU, for 256 compute units.  `own_rows` is their
# rule, `said_rows` what q_start says taken at its word, where rows that two
# requests name count twice.
def own_rows(q_start, T):
    ends = []
    for x in q_start:
        ends.append(max([min(max(x, 0), T), *ends[-1:]]))
    return [b - a for a, b in zip(ends, ends[1:])]


def said_rows(q_start, T):
    at = [min(max(x, 0), T) for x in q_start]
    return [max(b - a, 0) for a, b in zip(at, at[1:])]


def chunk_schedule(rows, lens, T, G, Hkv, mt=256, cus=256):
    """Pieces of work against the grid, split row tiles of pieces in the grid against
    those counted for the join, and the room for them and for their records."""
    target = 2 * cus if mt == 64 else cus
    tiles = [(-(-n * G // mt) if n * G > (16 if mt == 256 else 0) else 0, -(-max(L, 0) // 64))
             for n, L in zip(rows, lens)]
    C = max(4, -(-sum(a * b for a, b in tiles) * Hkv // target))
    splits = [max(1, (4 * b + C) // (4 * C)) if a else 0 for a, b in tiles]
    units = sum(a * k for (a, _), k in zip(tiles, splits)) * Hkv
    grid = (T * G // mt + len(rows)) * Hkv + target
    counted = sum(a for (a, _), k in zip(tiles, splits) if k > 1) * Hkv
    described, at = 0, 0
    for (a, _), k in zip(tiles, splits):
        for _ in range(a):
            described += sum(1 for h in range(Hkv) if at * Hkv + h < grid) if k > 1 else 0
            at += k
    records = sum(a * k for (a, _), k in zip(tiles, splits) if k > 1) * Hkv
    return dict(units=units, grid=grid, counted=counted, described=described, records=records,
                room=target)


def orders():
    """(q_start, lengths, T, G, Hkv, whether they need more than the grid has): rows
    that many requests name, the longest request last."""
    yield [0, 640] * 21, [64] * 40 + [32768], 640, 4, 1, True
    yield [0, 640] * 21, [64] * 40 + [32768], 640, 4, 8, True
    yield [0, 4096] * 50 + [0, 300], [64] * 100 + [32768], 4096, 4, 8, True
    yield [0, 300] + [100, 300] * 19 + [250, 640], [64] * 40 + [8000], 640, 4, 1, False


def test_rows_counted_twice_would_not_fit_the_grid():
    for q_start, lens, T, G, Hkv, too_many in orders():
        said = chunk_schedule(said_rows(q_start, T), lens, T, G, Hkv)
        assert (said["units"] > said["grid"]) is too_many
        assert (said["described"] < said["counted"]) is too_many
        own = chunk_schedule(own_rows(q_start, T), lens, T, G, Hkv)
        assert own["units"] <= own["grid"] and own["described"] == own["counted"]


def test_rows_counted_once_fit_the_grid():
    gen = torch.Generator().manual_seed(8)

    def below(n):
        return int(torch.randint(0, n, (1,), generator=gen))

    for turn in range(400):
        T, R, G, Hkv = 1 + below(5000), 1 + below(150), 1 + below(8), 1 + below(16)
        top = (2 ** below(12) + 2) * 64
        lens = [below(top) for _ in range(R)]
        q_start = [below(3 * T) - T for _ in range(R + 1)]
        if turn % 3 == 0:
            q_start.sort()
        for mt in (64, 256):
            s = chunk_schedule(own_rows(q_start, T), lens, T, G, Hkv, mt)
            assert s["units"] <= s["grid"] and s["described"] == s["counted"]
            assert s["counted"] <= s["room"] and s["records"] <= 2 * s["room"]


@pytest.mark.gpu
@pytest.mark.parametrize("q_start", [
    [0, 640] * 21, [0, 300] + [100, 300] * 19 + [250, 640],
    [0, 2 ** 31 - 1, -2 ** 31] * 13 + [5, 100, 2 ** 31 - 1]])
def test_attention_of_rows_that_many_requests_name(q_start):
    """Each row is the first request's that names it, and nothing around the output is
    written, also after calls of more rows whose splits stand in the workspace."""
    before = make_step([(3, 70), (900, 3000)], 4, 1, 64, 16, torch.float16, torch.float16)
    first = check_attention(before)
    s = make_step([(0, 64)] * 40 + [(0, 8000)], 4, 1, 64, 16, torch.float16, torch.float16,
                  extra=640)
    starts = [0]
    for n in own_rows(q_start, 640):
        starts.append(starts[-1] + n)
    want = attention_reference(s["q"], s["K"], s["V"], s["block_table"], ints(starts),
                               s["kv_len"], 1 / 8.0, True, None, None, None)
    around = torch.full((640 + 2 * 512, 4, 64), 7.0, dtype=torch.float16, device=DEV)
    s.update(q_start=ints(q_start), out=around[512:-512])
    for max_new in (None, 16, 1):
        around.fill_(7.0)
        check_attention(s, want=want, max_new=max_new)
        assert (around[:512] == 7.0).all() and (around[-512:] == 7.0).all()
    assert torch.equal(check_attention(before), first)


def test_lines_of_rows_counted_twice_would_pass_an_int():
    """The decode kernel's line of work: what the host bounds it by, and the tiles of
    16 keys of 2048 requests that name the same 4096 rows."""
    T, R, G, L, width = 4096, 4096, 4, 16384, 1024
    q_start = [0] + [0, T] * (R // 2)
    line = {rule: sum(-(-n * G // 16) * (L // 16) for n in rule(q_start, T))
            for rule in (said_rows, own_rows)}
    assert line[said_rows] >= 2 ** 31
    assert line[own_rows] <= (T * G // 16 + R) * (width + 1) < 2 ** 30


@pytest.mark.gpu
def test_attention_of_single_tokens_after_rows_that_many_requests_name():
    """Thousands of requests that name the same rows leave the kept workspace as
    they found it: calls that share it stay right."""
    T, R, G = 4096, 4096, 4
    fine = make_step([(1, 700 + 40 * r) for r in range(70)], G, 1, 64, 16, torch.float16,
                     torch.float16)
    first = check_attention(fine, max_new=1)
    s = make_step([(T, 8)], G, 1, 64, 16, torch.float16, torch.float16)
    table = torch.zeros(1, 1024, dtype=torch.int32, device=DEV)
    table[0, 0] = s["block_table"][0, 0]
    o, size = attention_reference(s["q"], s["K"], s["V"], table[:, :1], s["q_start"], s["kv_len"],
                                  1 / 8.0, True, None, None, None)
    s.update(block_table=table.expand(R, 1024), q_start=ints([0] + [T, 0] * (R // 2 - 1) + [T, T]),
             kv_len=ints([8] + [16384] * (R - 1)))
    check_attention(s, want=(o, size), max_new=1)
    assert torch.equal(check_attention(fine, max_new=1), first)


# -------------------------------------------------------------- a whole step
def run_step(state, freq, Hq):
    p = ops.paged_plan(state["past"], state["new"], state["table"], state["free"], 16,
                       state["qkv"].shape[0])
    q = ops.rope_append(state["qkv"], p.position, p.slot, state["K"], state["V"], freq)
    return p, q, ops.paged_attention(q, state["K"], state["V"], state["table"], p.q_start,
                                     p.kv_len)


def new_step(seed, past, new, pad=0, Hq=8, Hkv=2, D=64):
    gen = torch.Generator().manual_seed(seed)
    held = [-(-n // 16) for n in past]
    pages = sum(-(-(a + b) // 16) for a, b in zip(past, new)) + 4
    order = torch.randperm(pages, generator=gen).tolist()
    width = max(-(-(a + b) // 16) for a, b in zip(past, new))
    table, at = [], 0
    for n in held:
        table.append(order[at:at + n] + [-1] * (width - n))
        at += n
    K, V, *_ = cache_pair(gen, pages, Hkv, 16, D, torch.float16)
    return dict(past=ints(past), new=ints(new), table=ints(table), free=ints(order[at:]), K=K, V=V,
                qkv=torch.randn(sum(new) + pad, (Hq + 2 * Hkv) * D, generator=gen).half().to(DEV))


@pytest.mark.gpu
def test_a_step_of_all_three_against_64_bits():
    """Plan, append, attend: the new tokens' own keys are seen, rotary positions
    follow the plan's, and a second step goes on where the first one ended."""
    past, new = [40, 0, 17, 100], [1, 33, 0, 5]
    state = new_step(0, past, new, pad=3)
    freq = (10000.0 ** (-torch.arange(0, 64, 2) / 64)).to(DEV)
    for step in range(2):
        K0, V0 = state["K"].clone(), state["V"].clone()
        p, q, o = run_step(state, freq, 8)
        assert int(p.free_next) <= state["free"].numel()
        (yq, mq), (wk, mk), (wv, _) = rope_reference(state["qkv"], p.position, p.slot, K0, V0, freq,
                                                     2, None, False, None, None)
        u = HALF_STEP[torch.float16]
        assert ((q.double().cpu() - yq).abs() <= u * yq.abs() + 2.0 ** -20 * mq + 2.0 ** -25).all()
        assert ((state["K"].double().cpu() - wk).abs() <=
                u * wk.abs() + 2.0 ** -20 * mk + 2.0 ** -25).all()
        assert torch.equal(state["V"].double().cpu(), wv)
        s = dict(q=q, K=state["K"], V=state["V"], block_table=state["table"], q_start=p.q_start,
                 kv_len=p.kv_len, k_scale=None, v_scale=None)
        check_attention(s)
        state["past"] = p.kv_len.clone()
        state["new"] = ints([1, 1, 1, 1])
        state["free"] = state["free"][int(p.free_next):].contiguous()


@pytest.mark.gpu
def test_a_step_captured_and_replayed():
    """A captured step follows new lengths, inputs and tables on every replay, and
    two graphs replayed at once on two streams do not share a workspace."""
    freq = (10000.0 ** (-torch.arange(0, 64, 2) / 64)).to(DEV)
    cases = [([40, 0, 17], [1, 33, 2]), ([500, 30, 4], [30, 3, 3]), ([0, 900, 1], [1, 1, 34])]
    held = [new_step(i, past, new) for i, (past, new) in enumerate(cases)]
    pages = max(s["K"].shape[0] for s in held) + 60
    width = max(s["table"].shape[1] for s in held)

    def fill(live, s):
        for name in ("past", "new", "qkv"):
            live[name].copy_(s[name])
        live["table"].fill_(-1)
        live["table"][:, :s["table"].shape[1]] = s["table"]
        live["free"][:s["free"].numel()] = s["free"]
        for name in ("K", "V"):
            live[name][:s[name].shape[0]] = s[name]

    def fresh():
        gen = torch.Generator().manual_seed(99)
        K, V, *_ = cache_pair(gen, pages, 2, 16, 64, torch.float16)
        return dict(past=ints([0] * 3), new=ints([0] * 3), K=K, V=V,
                    table=torch.full((3, width), -1, dtype=torch.int32, device=DEV),
                    free=torch.arange(pages, dtype=torch.int32, device=DEV),
                    qkv=torch.zeros(36, 12 * 64, dtype=torch.float16, device=DEV))

    want = []
    for s in held:
        live = fresh()
        fill(live, s)
        want.append(run_step(live, freq, 8)[2].clone())
    lives, graphs, outs = [], [], []
    for _ in range(2):
        live = fresh()
        fill(live, held[0])
        run_step(live, freq, 8)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = run_step(live, freq, 8)[2]
        lives.append(live)
        graphs.append(g)
        outs.append(out)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for turn in range(6):
        which = [turn % 3, (turn + 1) % 3]
        for live, i in zip(lives, which):
            fill(live, held[i])
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                for _ in range(4):
                    g.replay()
        torch.cuda.synchronize()
        for out, i in zip(outs, which):
            assert torch.equal(out, want[i])
        run_step(fresh(), freq, 8)                    # eager work in between


@pytest.mark.gpu
def test_calls_at_once_on_two_streams():
    a = make_step([(1, 4000)], 8, 2, 128, 16, torch.float16, torch.float16)
    b = make_step([(1, 3000), (20, 900)], 8, 2, 128, 16, torch.float16, torch.float16, seed=1)
    want = [ops.paged_attention(**s) for s in (a, b)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, (s, st) in enumerate(zip((a, b), streams)):
            with torch.cuda.stream(st):
                got[i].append(ops.paged_attention(**s))
    torch.cuda.synchronize()
    for outs, w in zip(got, want):
        assert all(torch.equal(o, w) for o in outs)


@pytest.mark.gpu
def test_calls_of_threads_on_one_stream():
    """Threads that share a stream share its kept workspace; a call of three
    launches (single tokens, split chunks, their join) is not torn apart."""
    import threading

    steps = [make_step([(1, 900), (90, 4000 + 700 * i), (1, 70)], 6, 2, 128, 16, torch.float16,
                       torch.float16, seed=i) for i in range(4)]
    want = [check_attention(s) for s in steps]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        for _ in range(60):
            got = ops.paged_attention(**steps[i])
            if _ % 10 == 9 and not torch.equal(got, want[i]):
                bad.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    torch.cuda.synchronize()
    assert not bad


@pytest.mark.gpu
def test_native_call_path_and_python_steps_agree(monkeypatch):
    """The native call path takes these calls, and the Python steps give the same."""
    freq = (10000.0 ** (-torch.arange(0, 64, 2) / 64)).to(DEV)

    def step(fp8, wide):
        gen = torch.Generator().manual_seed(7)
        K, V, ks, vs = cache_pair(gen, 40, 2, 16, 64, FP8 if fp8 else torch.bfloat16, "tokens")
        table = torch.full((3, 9), -1, dtype=torch.int32, device=DEV)[:, :8]
        free = torch.arange(40, dtype=torch.int32, device=DEV)
        p = ops.paged_plan(ints([0, 0, 0]), ints([30, 1, wide]), table, free, 16, 31 + wide,
                           free_start=ints([2]))
        qkv = torch.randn(31 + wide, 8 * 64, generator=gen).bfloat16().to(DEV)
        q = ops.rope_append(qkv, torch.stack([p.position, p.position + 3]), p.slot, K, V, freq,
                            axes=[0] * 10 + [1] * 22, interleaved=fp8, k_scale=ks, v_scale=vs)
        o = [ops.paged_attention(q, K, V, table, p.q_start, p.kv_len, k_scale=ks, v_scale=vs, **kw)
             for kw in ({}, dict(max_new=30, window=9), dict(causal=False, scale=0.2),
                        dict(max_new=1))]
        return [*p, q, K.view(torch.uint8) if fp8 else K, V.view(torch.uint8) if fp8 else V, *o]

    assert ops._fast is not None
    for fp8, wide in ((False, 1), (True, 70)):
        step(fp8, wide)                                  # makes the workspaces
        calls = []
        with monkeypatch.context() as m:
            class Watch:
                def __getattr__(self, name):
                    fn = getattr(fast, name)

                    def call(*args):
                        r = fn(*args)
                        calls.append((name, r is not None))
                        return r
                    return call

            fast = ops._fast
            m.setattr(ops, "_fast", Watch())
            native = step(fp8, wide)
        assert len(calls) == 6 and all(took for _, took in calls), calls
        with monkeypatch.context() as m:
            m.setattr(ops, "_fast", None)
            steps = step(fp8, wide)
        for a, b in zip(native, steps):
            assert a.dtype == b.dtype and torch.equal(a, b)


# ------------------------------------------------------------------- refusals
P = 0x10000  # a fake, aligned device address: never dereferenced


@pytest.fixture(scope="module")
def lib():
    from decodebench_amd import build

    if not ops.LIB_PATH.exists():
        build.build(verbose=False)
    return ops.load_library()


def last(lib):
    return lib.db_last_error().decode()


def a_cache(**kw):
    c = dict(k=P, v=P, k_scale=None, v_scale=None, k_page_stride=16384, k_head_stride=2048,
             k_token_stride=128, v_page_stride=16384, v_head_stride=2048, v_token_stride=128,
             pages=10, page_size=16, Hkv=8, D=128, dtype=0)
    return ops._PagedCache(**{**c, **kw})


def test_plan_contract_errors(lib):
    ok = dict(past=P, fresh=P, table=P, stride=8, width=8, free=P, count=9, start=None, page=16, R=2,
              T=4, q=P, kv=P, pos=P, slot=P, nxt=P)

    def call(**kw):
        return lib.db_paged_plan(*{**ok, **kw}.values(), None)

    for bad in (dict(R=-1), dict(T=-1), dict(count=-1), dict(width=0), dict(page=0),
                dict(stride=7), dict(past=None), dict(table=None), dict(slot=None), dict(q=None),
                dict(nxt=None), dict(free=None), dict(past=P + 2), dict(slot=P + 4)):
        assert call(**bad) == -1, bad
        assert "db_paged_plan" in last(lib)


def test_rope_contract_errors(lib):
    ok = dict(qkv=P, stride=48 * 128, position=P, n_axes=1, axes=None, slot=P, freq=P, rot=128,
              inter=0, cache=a_cache(), q=P, T=3, Hq=32, dtype=0)

    def call(**kw):
        a = {**ok, **kw}
        a["cache"] = C.byref(a["cache"])
        return lib.db_rope_append(*a.values(), None)

    for bad in (dict(T=-1), dict(Hq=0), dict(rot=8), dict(rot=144), dict(rot=120), dict(n_axes=0),
                dict(n_axes=5), dict(stride=48 * 128 - 8), dict(stride=48 * 128 + 4),
                dict(qkv=None), dict(slot=None), dict(q=None), dict(freq=None), dict(qkv=P + 8),
                dict(position=P + 2), dict(slot=P + 4), dict(dtype=1), dict(dtype=2), dict(dtype=7),
                dict(n_axes=2, axes=bytes([0] * 63 + [2])),
                dict(cache=a_cache(k=None)), dict(cache=a_cache(D=120)), dict(cache=a_cache(D=272)),
                dict(cache=a_cache(pages=0)), dict(cache=a_cache(page_size=0)),
                dict(cache=a_cache(Hkv=0)), dict(cache=a_cache(k_token_stride=4)),
                dict(cache=a_cache(v_page_stride=-8)), dict(cache=a_cache(v=P + 8)),
                dict(cache=a_cache(k_scale=P)), dict(cache=a_cache(dtype=1)),
                dict(cache=a_cache(dtype=1, k_scale=P, v_scale=P + 2)),
                dict(cache=a_cache(dtype=1, k_scale=P, v_scale=P, k_token_stride=136)),
                dict(cache=a_cache(dtype=5))):
        assert call(**bad) == -1, bad
        assert "db_rope_append" in last(lib)


def test_attention_contract_errors(lib):
    ok = dict(q=P, qt=4096, qh=128, o=P, cache=a_cache(), table=P, stride=8, width=8, start=P, kv=P,
              T=4, R=2, Hq=32, most=0, scale=0.1, causal=1, window=0, dtype=0, ws=P,
              bytes=1 << 40)

    def call(**kw):
        a = {**ok, **kw}
        a["cache"] = C.byref(a["cache"])
        return lib.db_paged_attention(*a.values(), None)

    for bad in (dict(T=-1), dict(R=-1), dict(Hq=30), dict(Hq=0), dict(most=-1), dict(scale=0.0),
                dict(scale=-1.0), dict(scale=math.inf), dict(scale=math.nan), dict(window=-1),
                dict(window=4, causal=0), dict(width=0), dict(stride=-1), dict(qt=4092),
                dict(qh=-128), dict(q=None), dict(o=None), dict(table=None), dict(start=None),
                dict(kv=None), dict(q=P + 8), dict(o=P + 2), dict(table=P + 1), dict(ws=None),
                dict(ws=P + 16), dict(dtype=2), dict(T=2 ** 27, Hq=32),
                dict(cache=a_cache(D=256)), dict(cache=a_cache(D=96)),
                dict(cache=a_cache(dtype=1)), dict(cache=a_cache(pages=-1))):
        assert call(**bad) == -1, bad
        assert "db_paged_attention" in last(lib)
    assert call(cache=a_cache(D=96)) == -1 and "64 and 128" in last(lib)


def test_paged_calls_too_large_are_refused(lib):
    """Sizes whose tiles, rows or grids an int could not count."""
    far = 2 ** 27
    cache = a_cache(k_page_stride=16384, v_page_stride=16384)
    for T, R, Hq, most, width in (
            (4, 8, 32, 1, far), (4, 64, 32, 1, far // 8), (4, 8, 32, 0, far),   # key tiles of all
            (2 ** 24, 1, 32, 1, 256), (4, 1, 32, 1, 2 ** 30),                   # ... row tiles too
            (2 ** 25, 4, 32, 0, 8), (4, 2 ** 19, 32, 1, 8)):                    # rows, requests
        assert lib.db_paged_attention(P, 4096, 128, P, C.byref(cache), P, width, width, P, P, T, R,
                                      Hq, most, 0.1, 1, 0, 0, P, 1 << 40, None) == -1, (T, R, width)
        assert "too large" in last(lib)
    for T, R, count in ((2 ** 30 + 1, 2, 9), (4, 2 ** 30 + 1, 9), (4, 2, 2 ** 30 + 1)):
        assert lib.db_paged_plan(P, P, P, 8, 8, P, count, None, 16, R, T, P, P, P, P, P, None) == -1
        assert "above" in last(lib)
    assert lib.db_rope_append(P, 48 * 128, P, 1, None, P, P, 128, 0, C.byref(a_cache()), P, 2 ** 26,
                              32, 0, None) == -1 and "2^26" in last(lib)


def test_rope_append_refuses_a_cache_whose_rows_share_memory(lib):
    for bad in ("k_page_stride", "v_page_stride", "k_head_stride", "v_head_stride",
                "k_token_stride", "v_token_stride"):
        assert lib.db_rope_append(P, 48 * 128, P, 1, None, P, P, 128, 0,
                                  C.byref(a_cache(**{bad: 0})), P, 3, 32, 0, None) == -1, bad
        assert "share memory" in last(lib)


def test_paged_workspace_of_refused_calls_is_none(lib):
    f = lib.db_paged_attention_workspace_bytes
    for bad in ((0, 32, 8, 128, 1, 1), (1, 30, 8, 128, 1, 1), (1, 32, 8, 96, 1, 1),
                (1, 32, 8, 128, 0, 1), (1, 32, 8, 128, 1, -1)):
        assert f(*bad, None) == 0


def test_paged_wrappers_refuse_cpu_tensors():
    x, i = torch.zeros(2, 6 * 64, dtype=torch.float16), torch.zeros(2, dtype=torch.int32)
    K = torch.zeros(4, 2, 16, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="GPU"):
        ops.paged_plan(i, i, torch.zeros(2, 3, dtype=torch.int32), i, 16, 2)
    with pytest.raises(ValueError, match="GPU"):
        ops.rope_append(x, i, i.long(), K, K, torch.ones(32))
    with pytest.raises(ValueError, match="GPU"):
        ops.paged_attention(x.view(2, 6, 64), K, K, i.view(2, 1), i, i)


@pytest.mark.gpu
def test_paged_wrappers_refuse():
    s = make_step([(2, 20), (1, 9)], 4, 2, 64, 16, torch.float16, torch.float16)

    def attention(**kw):
        return ops.paged_attention(**{**s, **kw})

    for exc, kw in (
            (TypeError, dict(q=s["q"].float())), (TypeError, dict(q=s["q"].bfloat16())),
            (TypeError, dict(q_start=s["q_start"].long())),
            (ValueError, dict(q=s["q"][0])), (ValueError, dict(q=s["q"][:, :3])),
            (ValueError, dict(q=s["q"].transpose(1, 2))), (ValueError, dict(kv_len=ints([1]))),
            (ValueError, dict(q_start=ints([0, 1]))), (ValueError, dict(window=0)),
            (ValueError, dict(window=3, causal=False)), (ValueError, dict(max_new=0)),
            (ValueError, dict(scale=-0.5)), (ValueError, dict(scale=0.0)),
            (ValueError, dict(k_scale=torch.ones(2, device=DEV))),
            (ValueError, dict(V=s["V"][:1])), (ValueError, dict(K=s["K"][:0], V=s["V"][:0])),
            (ValueError, dict(K=s["K"].to(FP8), V=s["V"].to(FP8))),
            (ValueError, dict(K=s["K"].to(FP8), V=s["V"].to(FP8),
                              k_scale=torch.ones(3, device=DEV), v_scale=torch.ones(2, device=DEV))),
            (ValueError, dict(out=torch.empty(3, 4, 32, device=DEV).half())),
            (TypeError, dict(out=torch.empty(3, 4, 64, device=DEV)))):
        with pytest.raises(exc):
            attention(**kw)
    qkv = torch.zeros(3, 8 * 64, dtype=torch.float16, device=DEV)
    slot = ints([0, 1, 2], torch.int64)
    freq = torch.ones(32, device=DEV)
    args = dict(qkv=qkv, position=ints([0, 1, 2]), slot=slot, K=s["K"], V=s["V"], inv_freq=freq)
    for exc, kw in (
            (ValueError, dict(qkv=qkv[:, :-8])), (ValueError, dict(qkv=qkv[:, :4 * 64])),
            (ValueError, dict(position=ints([0, 1]))), (TypeError, dict(slot=slot.int())),
            (ValueError, dict(position=ints([[0, 1, 2]] * 3))),
            (ValueError, dict(position=ints([[0, 1, 2]] * 2), axes=[0] * 31 + [2])),
            (ValueError, dict(axes=[0] * 31)), (ValueError, dict(inv_freq=freq[:31])),
            (ValueError, dict(inv_freq=torch.ones(48, device=DEV))),
            (TypeError, dict(inv_freq=freq.double()))):
        with pytest.raises(exc):
            ops.rope_append(**{**args, **kw})
    table = ints([[0, 1], [2, 3]])
    plan = dict(past_len=ints([1, 2]), new_len=ints([1, 1]), block_table=table,
                free_pages=ints([5]), page_size=16, n_tokens=2)
    for exc, kw in (
            (ValueError, dict(past_len=ints([1]))), (TypeError, dict(new_len=ints([1, 1]).long())),
            (ValueError, dict(page_size=0)), (ValueError, dict(n_tokens=-1)),
            (ValueError, dict(page_size=2 ** 32 + 16)), (ValueError, dict(n_tokens=2 ** 32 + 2)),
            (ValueError, dict(block_table=table[:1].expand(2, 2))),
            (ValueError, dict(block_table=table.t())),
            (ValueError, dict(free_pages=table)), (ValueError, dict(free_start=ints([0, 1])))):
        with pytest.raises(exc):
            ops.paged_plan(**{**plan, **kw})
