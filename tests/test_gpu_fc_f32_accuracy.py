"""fp32 FullConnect layers have the accuracy of fp32, not of two bf16 planes, on every route.

Relative 2-norm errors of products of N(0, 1) matrices over K terms.  Sums of K independent terms and of K independent errors both grow with sqrt(K), so an error of e of every
product is one of e of the result: 2^-24 for the products of planes that are dropped (m l, l m, l l), 2^-24 for the output's rounding, 2^-24 sqrt(K / 64) for the running sums.  The
tensor core truncates, by up to 2^-23 of an accumulator an instruction: four into the hh accumulator of a window of 64 terms, 2^-21 of the window's sum, of any sign
against the others; and 5 K / 16 into the accumulator of the side products, which are 2^-7 of the sum at most."""
import pytest

torch = pytest.importorskip("torch")


def bound(K):
    return 2.0 ** -24 * (2 + (K / 64) ** 0.5) + 2.0 ** -21 + 5 * K / 16 * 2.0 ** -23 * 2.0 ** -7


def planes(x):
    """fp32 as three bf16 words, in 64 bits."""
    h = x.bfloat16()
    m = (x - h.float()).bfloat16()
    l = (x - h.float() - m.float()).bfloat16()
    return h.double(), m.double(), l.double()


@pytest.mark.parametrize("K", (64, 300, 512))
def test_the_bound_tells_a_lost_product(K):
    """On the CPU: without either of the six products of planes the error is past the bound, with all of them well within."""
    gen = torch.Generator().manual_seed(K)
    a, b = torch.randn(60, K, generator=gen), torch.randn(K, 70, generator=gen)
    ref = a.double() @ b.double()
    x, y = planes(a), planes(b)
    kept = [(0, 0), (0, 1), (1, 0), (1, 1), (0, 2), (2, 0)]
    error = lambda pairs: float((sum(x[i] @ y[j] for i, j in pairs) - ref).norm() / ref.norm())
    assert error(kept) <= 2.0 ** -24
    for lost in kept:
        assert error([p for p in kept if p != lost]) > 1.2 * bound(K), lost


@pytest.fixture(scope="module")
def eng(pkg):
    return pkg.submodule("engine").Engine()


@pytest.fixture(scope="module")
def lib(pkg):
    return pkg.submodule("lib")


# rows, option, what the plan says
ROUTES = [(1, 0, "small"), (2, 0, "small"), (4, 0, "small"), (301, 2, "planes 128x"), (301, 1, "pair 256x256"), (301, 11, "pair 256x128")]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,tile,plan", ROUTES)
@pytest.mark.parametrize("IC", (64, 300, 512))
def test_forward(eng, lib, rows, tile, plan, IC):
    gen = torch.Generator(device="cuda").manual_seed(rows)
    X, W = torch.randn(rows, IC, device="cuda", generator=gen), torch.randn(600, IC, device="cuda", generator=gen)
    old = lib.set_option("FC_TILE", tile)
    try:
        z = X.double() @ W.double().T
        Y = eng.fullConnect(X, W)
        assert plan in lib.last_plan(), lib.last_plan()
        assert float((Y - z).norm() / z.norm()) <= bound(IC)
        _, Z = eng.fullConnect_glu(X, W, save=True)
        assert plan in lib.last_plan(), lib.last_plan()
        assert float((Z - z).norm() / z.norm()) <= bound(IC)
    finally:
        lib.set_option("FC_TILE", old)
    assert lib.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("tile,plan", [r[1:] for r in ROUTES[3:]])
@pytest.mark.parametrize("rows,IC,OC", [(64, 260, 64), (300, 512, 256), (512, 132, 512), (500, 1000, 77)])
@pytest.mark.parametrize("glu", (False, True), ids=("fc", "glu"))
def test_gradients(eng, lib, tile, plan, rows, IC, OC, glu):
    gen = torch.Generator(device="cuda").manual_seed(OC)
    if glu:
        OC //= 2
    H = 2 if glu else 1
    X, W, dY = torch.randn(rows, IC, device="cuda", generator=gen), torch.randn(H * OC, IC, device="cuda", generator=gen), torch.randn(rows, OC, device="cuda", generator=gen)
    old = lib.set_option("FC_TILE", tile)
    try:
        if glu:                                   # U = G = 1 and no activation: both halves of deltaZ are deltaY
            dX, dW, _ = eng.fullConnect_glu_delta(dY, X, W, torch.ones(rows, 2 * OC, device="cuda"), act="none")
            dY = torch.cat([dY, dY], 1)
        else:
            dX, dW, _ = eng.fullConnect_delta(dY, X, W)
        assert plan in lib.last_plan(), lib.last_plan()
    finally:
        lib.set_option("FC_TILE", old)
    for got, a, b in ((dX, dY, W), (dW, dY.T, X)):
        ref = a.double() @ b.double()
        assert float((got - ref).norm() / ref.norm()) <= bound(a.shape[1])
    assert lib.device_status() == 0
