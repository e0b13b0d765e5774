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
