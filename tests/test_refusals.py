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
