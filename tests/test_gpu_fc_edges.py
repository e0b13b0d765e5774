"""FullConnect layers at the ends of their ranges: sizes, values, scratch, and what the operators hand to one another."""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng(pkg):
    return pkg.submodule("engine").Engine()


@pytest.fixture(scope="module")
def lib(pkg):
    return pkg.submodule("lib")


def test_residual_of_2_28_columns(eng, lib):
    """Rows of the residual that lie 2^32 bytes and more apart.  Sums and residual are small whole numbers, exact in bf16; W repeats, so that rows of Y
    are compared by parts."""
    rows, OC, some = 17, 1 << 28, 1 << 16
    gen = torch.Generator(device="cuda").manual_seed(1)
    X = torch.randint(-2, 3, (rows, 8), device="cuda", generator=gen).bfloat16()
    W = torch.randint(-2, 3, (some, 8), device="cuda", generator=gen).bfloat16()
    z = X.float() @ W.float().T                                     # (at most 32)
    R = torch.empty(rows, OC, device="cuda", dtype=torch.bfloat16)
    for r in range(rows):
        R[r] = 64 + r
    Y = eng.fullConnect(X, W.repeat(OC // some, 1), Residual=R)
    del R
    want = z + 64 + torch.arange(rows, device="cuda")[:, None]
    Y = Y.view(rows, OC // some, some)
    for r in range(rows):
        assert (Y[r].float() == want[r]).all(), r
    assert lib.device_status() == 0


def test_f32_runs_without_scratch_where_the_card_is_full(eng, lib):
    """Operands split once need 157 MB of scratch; where cudaMalloc refuses it the products are gathered, as they are in a capture."""
    gen = torch.Generator(device="cuda").manual_seed(2)
    rows, IC, OC = 8192, 2048, 2048
    X, dY = torch.randn(rows, IC, device="cuda", generator=gen), torch.randn(rows, OC, device="cuda", generator=gen)
    W = torch.randn(OC, IC, device="cuda", generator=gen) * IC ** -0.5
    Y, Z, dZ, dX, dW, dB = (torch.empty_like(t) for t in (dY, dY, dY, X, W, W[0]))
    plans = []

    def step():
        eng.base.fullConnect(Y, X, W, rows, IC, OC, 0, lib.ACTS["silu"], 0.0, None, None, Z)
        plans.append(lib.last_plan())
        eng.base.fullConnect_delta(dX, dW, dB, dY, X, W, Z, dZ, rows, IC, OC, 0, lib.ACTS["silu"], 0.0)
        plans.append(lib.last_plan())

    step()                                          # (kernels take memory when they are first used: both routes once)
    old = lib.set_option("FC_TILE", 2)
    try:
        step()
    finally:
        lib.set_option("FC_TILE", old)
    torch.cuda.synchronize()
    want = [t.clone() for t in (Y, Z, dX, dW, dB)]
    for t in (Y, Z, dX, dW, dB):
        t.fill_(float("nan"))
    lib.release_workspace()
    torch.cuda.empty_cache()
    free, _ = torch.cuda.mem_get_info()
    hog = torch.empty(free - (100 << 20), dtype=torch.uint8, device="cuda")
    try:
        with torch.cuda.stream(torch.cuda.Stream()):
            step()
        torch.cuda.synchronize()
    finally:
        del hog
        torch.cuda.empty_cache()
    assert "pair" in plans[0] and "pair" in plans[1], plans
    assert "planes 128x" in plans[4] and "planes 128x" in plans[5], plans
    # sums of K terms with deviation sqrt(K): either way within a few 2^-23 of that
    for got, ref in zip((Y, Z, dX, dW, dB), want):
        assert float((got - ref).norm() / ref.norm()) <= 2.0 ** -20
    assert lib.device_status() == 0
