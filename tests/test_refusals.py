"""Refusals of the C ABI that hold with and without a GPU, and the ones that may only
be tried without."""

import conftest
import pytest

torch = pytest.importorskip("torch")

from decodebench_amd import ops  # noqa: E402

P = 0x10000  # a fake, 256-byte aligned device address: never dereferenced


@pytest.fixture(scope="module")
def lib():
    from decodebench_amd import build

    if not ops.LIB_PATH.exists():
        build.build(verbose=False)
    return ops.load_library()


class Item:
    def __init__(self, name, *keywords):
        self.name, self.keywords, self.skipped = name, keywords, False

    def add_marker(self, mark):
        self.skipped = mark.name == "skip"


@pytest.mark.parametrize("gpu", [False, True])
def test_calls_that_a_gpu_would_take_stay_off_it(gpu, monkeypatch):
    monkeypatch.setattr(conftest, "_has_gpu", lambda: gpu)
    items = [Item("test_gemm_contract"), Item("test_quantize_contract"), Item("test_gemm", "gpu")]
    conftest.pytest_collection_modifyitems(None, items)
    assert [i.skipped for i in items] == [gpu, False, not gpu]


def test_gemm_needs_its_workspace(lib):
    """Forty tokens are quantised in a launch of their own, whatever the GPU."""
    def call(work=P, nbytes=1 << 24, xs=None):
        return lib.db_gemm_blocks(P, 256, xs, 0, 0, P, P, P, 40, 256, 64, 0, 0, work, nbytes, None)

    for bad in (dict(work=None), dict(work=P + 128), dict(nbytes=256), dict(xs=P)):
        assert call(**bad) == ops.DB_ERR_INVALID, bad
        assert b"db_gemm_blocks" in lib.db_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("B", [1, 4, 40])
def test_projections_do_not_write_over_x(B):
    """Every workgroup reads all of x, some after others have written their outputs."""
    K = 256
    gen = torch.Generator().manual_seed(B)
    buf = torch.randn(2 * B, K, generator=gen).half().cuda()
    x, g = buf[:B], torch.ones(K).half().cuda()
    W, W2 = ((torch.randn(K, K, generator=gen) / 16).half().cuda() for _ in range(2))
    before = buf.clone()
    for call in (lambda out: ops.gemv(x, W, out=out), lambda out: ops.f1_rmsnorm_gemv(x, g, W, out=out),
                 lambda out: ops.f2_gateup_swiglu(x, W, W2, out=out),
                 lambda out: ops.f2_rmsnorm_gateup_swiglu(x, g, W, W2, out=out)):
        with pytest.raises(ValueError, match="share memory with x"):
            call(x)
        assert torch.equal(buf, before)
        beside = torch.empty_like(x)
        want = call(beside).clone()
        assert torch.equal(call(buf[B:]), want)
        buf.copy_(before)


def a_layer(**more):
    m = dict(wg=P, wu=P, wd=P, sg=None, su=None, sd=None, E=4, H=16, I=2048, dtype=0, w_dtype=0)
    m.update(more)
    return ops._Moe(*(m[f[0]] for f in ops._Moe._fields_))


def test_workspace_of_refused_calls_is_none(lib):
    """What an entry point refuses for its sizes asks for no workspace first."""
    for sizes in (dict(m=a_layer(), T=1 << 19, k=64), dict(m=a_layer(H=1 << 19, I=16), T=64, k=16),
                  dict(m=a_layer(I=2044), T=4, k=2), dict(m=a_layer(H=12), T=4, k=2),
                  dict(m=a_layer(w_dtype=1, I=2056), T=4, k=2), dict(m=a_layer(dtype=1), T=4, k=2),
                  dict(m=a_layer(w_dtype=2), T=4, k=2), dict(m=a_layer(), T=4, k=65)):
        m, T, k = sizes.values()
        assert lib.db_moe_experts_workspace_bytes(m, T, k) == 0, (m.H, m.I, T, k)
        assert lib.db_moe_layer_workspace_bytes(m, T, k) == 0
        assert lib.db_moe_experts(P, m.H, P, P, m, P, T, k, None, 0, None) == ops.DB_ERR_INVALID
        assert b"workspace" not in lib.db_last_error()
    m = a_layer()
    assert lib.db_moe_layer_workspace_bytes(m, 4, 5) == 0       # five of four experts
    assert lib.db_moe_experts_workspace_bytes(m, 4, 5) > 0
    # the largest calls, and what the experts take
    for T, k, H, I in ((1 << 18, 1, 16, 2032), (4, 64, 64, 64)):
        m = a_layer(H=H, I=I)
        assert lib.db_moe_experts_workspace_bytes(m, T, k) >= T * k * (2 * I + 4 * H)
    for T, H, E in ((4, 12, 8), (4, 4, 8), (1 << 20, 64, 8), (4, 64, 1025)):
        assert lib.db_moe_route_workspace_bytes(T, H, E) == 0
    for T, K, N, dtype in ((40, 40, 64, 0), (40, 8, 64, 0), (40, 64, 64, 7), (1 << 22, 64, 64, 0)):
        assert lib.db_gemm_blocks_workspace_bytes(T, K, N, dtype) == 0


@pytest.mark.gpu
def test_too_many_tokens_are_refused_before_memory_is_taken():
    T, k, H, I = 1 << 19, 64, 16, 2048
    x = torch.zeros(T, H, dtype=torch.float16, device="cuda")
    Wg, Wd = (torch.zeros(1, *s, dtype=torch.float16, device="cuda") for s in ((I, H), (H, I)))
    e = torch.zeros(T, k, dtype=torch.int32, device="cuda")
    w = torch.zeros(T, k, device="cuda")
    torch.cuda.reset_peak_memory_stats()
    start = torch.cuda.memory_allocated()
    with pytest.raises(ValueError, match="too many"):
        ops.moe_experts(x, e, w, Wg, Wg, Wd)
    assert torch.cuda.max_memory_allocated() - start <= 2 * x.numel() * 2
    Wr = torch.zeros(1024, H, dtype=torch.float16, device="cuda")
    torch.cuda.reset_peak_memory_stats()
    with pytest.raises(ValueError, match="top_k"):
        ops.moe_route(x, Wr, 65)
    assert torch.cuda.max_memory_allocated() - start <= 2 * Wr.numel()
