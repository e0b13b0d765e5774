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


# ---- fp32 products: operands of every magnitude, without a cost for the ordinary ones beside them ----

PAIRS = pytest.mark.parametrize("tile", (1, 11, 2), ids=("pairs", "pairs of 128 columns", "gathered"))


@pytest.fixture
def tiled(lib):
    held = []

    def set_tile(tile):
        held.append(lib.set_option("FC_TILE", tile))
    yield set_tile
    for old in reversed(held):
        lib.set_option("FC_TILE", old)
    assert lib.device_status() == 0, lib.last_error()


def near(got, a, b):
    """got = a b: (K / 16 + 8) 2^-22 of the sum of magnitudes (hh accumulators truncate, at most 2^-23 of a product is dropped), an output's rounding, and the last place of a
    denormal, 2^-149, in each product and sum."""
    K = a.shape[1]
    ref, S = a.double() @ b.double(), a.double().abs() @ b.double().abs()
    bad = ~((got.double() - ref).abs() <= (K / 16 + 8) * 2.0 ** -22 * S + 2.0 ** -24 * ref.abs() + K * 2.0 ** -148)
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist())


def powers(n):
    """2^0 ... 2^-148, n of them."""
    return torch.exp2(-torch.linspace(0, 148, n, dtype=torch.float64, device="cuda"))


def of_magnitudes(gen, what, m, n):
    t = torch.randn(m, n, device="cuda", generator=gen, dtype=torch.float64)
    if what == "rows":
        t *= powers(m)[:, None]
    elif what == "columns":
        t *= powers(n)
    elif what == "elements":
        t *= torch.exp2(-torch.randint(0, 149, (m, n), device="cuda", generator=gen).double())
    return t.float()


@PAIRS
@pytest.mark.parametrize("first,second", [("rows", ""), ("columns", ""), ("elements", ""), ("", "rows"), ("", "columns"), ("", "elements"), ("rows", "rows"), ("elements", "elements")])
def test_f32_of_every_magnitude(eng, tiled, tile, first, second):
    gen = torch.Generator(device="cuda").manual_seed(3)
    tiled(tile)
    rows, IC, OC = 301, 204, 149
    X, W, V, dY = of_magnitudes(gen, first, rows, IC), of_magnitudes(gen, second, OC, IC), of_magnitudes(gen, second, 2 * OC, IC), of_magnitudes(gen, first, rows, OC)
    near(eng.fullConnect(X, W), X, W.T)
    near(eng.fullConnect_glu(X, V, act="none", save=True)[1], X, V.T)
    dX, dW, _ = eng.fullConnect_delta(dY, X, W)
    near(dX, dY, W)
    near(dW, dY.T, X)
    # (gates and ups of deltaZ: act 'none' and U = G = 1 make both of them deltaY)
    one = torch.ones(rows, 2 * OC, device="cuda")
    dX, dV, _ = eng.fullConnect_glu_delta(dY, X, V, one, act="none")
    both = torch.cat([dY, dY], 1)
    near(dX, both, V)
    near(dV, both.T, X)


@PAIRS
@pytest.mark.parametrize("everywhere", (True, False))
def test_f32_rows_and_columns_of_zeros_beside_tiny_elements(eng, tiled, tile, everywhere):
    """`everywhere`: a column of X and of W holds denormals, in the rows that are zero otherwise too."""
    gen = torch.Generator(device="cuda").manual_seed(4)
    tiled(tile)
    rows, IC, OC = 520, 300, 260
    X, W, dY = of_magnitudes(gen, "", rows, IC), of_magnitudes(gen, "", OC, IC), of_magnitudes(gen, "", rows, OC)
    X[::3], W[::5], dY[:, ::7] = 0, 0, 0
    X[1, 5] = W[2, 9] = dY[4, 8] = 1e-36
    if everywhere:
        X[:, 11] = W[:, 12] = 3e-40
    Y = eng.fullConnect(X, W)
    near(Y, X, W.T)
    zero = (X.double().abs() @ W.double().abs().T) == 0
    assert bool(zero[::3].all()) != everywhere and not Y[zero].any()
    dX, dW, _ = eng.fullConnect_delta(dY, X, W)
    near(dX, dY, W)
    near(dW, dY.T, X)
    assert not dW[::7].any()


@PAIRS
def test_f32_infinite_beside_tiny_elements(eng, tiled, tile):
    """What an Inf meets is Inf or NaN as in 64 bits, its neighbours in a word keep their values."""
    gen = torch.Generator(device="cuda").manual_seed(5)
    tiled(tile)
    rows, IC, OC = 300, 200, 136
    X, W = of_magnitudes(gen, "", rows, IC), of_magnitudes(gen, "", OC, IC)
    X[7, 20], X[7, 21], X[8, 21], X[9, 22], X[40, 23] = float("inf"), 1e-36, 1e-37, 3.4e38, float("nan")
    W[:, 20:24] *= 2.0 ** -20
    Y = eng.fullConnect(X, W)
    ref = X.double() @ W.double().T
    assert torch.equal(torch.isnan(Y), torch.isnan(ref)) and torch.equal(torch.isinf(Y), torch.isinf(ref))
    fine = torch.ones(rows, dtype=torch.bool, device="cuda")
    fine[7] = fine[40] = False
    near(Y[fine], X[fine], W.T)


def test_f32_softmax_tails_cost_little(eng, lib):
    """deltaY of a classifier whose softmax has tails of 1e-30 to 1e-45: the sums it goes into are ordinary, and are not formed once more.  They
    took 53 times as long as without."""
    gen = torch.Generator(device="cuda").manual_seed(6)
    rows, IC, OC = 512, 4096, 1000
    X, W = torch.randn(rows, IC, device="cuda", generator=gen), torch.randn(OC, IC, device="cuda", generator=gen) * IC ** -0.5
    logits = torch.randn(rows, OC, device="cuda", generator=gen)
    times = []
    for sharp in (1, 40):
        dY = torch.softmax(logits * sharp, 1)
        assert bool(((dY > 0) & (dY < 1e-33)).any()) == (sharp > 1)
        best = 1e9
        for _ in range(10):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            dX, dW, _ = eng.fullConnect_delta(dY, X, W)
            b.record()
            b.synchronize()
            best = min(best, a.elapsed_time(b))
        assert "pair" in lib.last_plan()
        times.append(best)
        near(dX, dY, W)
        near(dW, dY.T, X)
    assert times[1] <= 5 * times[0], times


def test_f32_long_reductions_on_few_sms(eng, lib):
    """Two tiles in turn on one pair, 2.2 million steps each: should the sums of the first have to be formed once more, the second could wait too long.  They are cut, or gathered."""
    rows, IC, OC = 257, 2200000, 128
    gen = torch.Generator(device="cuda").manual_seed(7)
    X, W = torch.randn(rows, IC, device="cuda", generator=gen), torch.randn(OC, IC, device="cuda", generator=gen)
    old = lib.set_option("SM_BUDGET", 2)
    try:
        Y = eng.fullConnect(X, W)
        plan = lib.last_plan()
        assert "planes 128x" in plan or int(plan.split("parts=")[1]) > 1, plan
    finally:
        lib.set_option("SM_BUDGET", old)
    some = torch.tensor([0, 100, 255, 256], device="cuda")
    near(Y[some], X[some], W.T)
    eng.fullConnect(X, W)
    assert lib.device_status() == 0


# ---- activations at the ends of their range ----

ROUTES = [("f32", 2, 0), ("f32", 70, 2), ("f32", 70, 1), ("bf16", 2, 0), ("bf16", 70, 0), ("f16", 2, 0), ("f16", 70, 1)]
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def through_act(eng, tiled, dtype, rows, tile, act, k, values):
    """act of `values` (at most 8), the same by the gated block (U = 1), and both gradients of deltaY = 1; rows x 8 each, the values as columns.  W takes
    them through unchanged: X is 1 in its first column and 0 behind, W has them as its first column."""
    t = TYPES[dtype]
    tiled(tile)
    z = torch.tensor(values, device="cuda").to(t)
    X = torch.zeros(rows, 8, device="cuda", dtype=t)
    X[:, 0] = 1
    bias = torch.zeros(8, device="cuda", dtype=t)
    bias[:len(values)] = z                          # (by the bias: an Inf in W would meet zeros)
    W = torch.zeros(8, 8, device="cuda", dtype=t)
    y = eng.fullConnect(X, W, bias, act=act, k=k)
    g = eng.fullConnect_glu(X, torch.zeros(16, 8, device="cuda", dtype=t), torch.cat([bias, torch.ones_like(bias)]), act=act, k=k)
    Z = bias.expand(rows, 8).contiguous()
    one = torch.ones(rows, 8, device="cuda", dtype=t)
    # deltaB sums a column's rows: of one row it is deltaZ itself
    slope = eng.fullConnect_delta(one[:1], X[:1], W, Z[:1], act=act, k=k, bias=True)[2]
    both = eng.fullConnect_glu_delta(one[:1], X[:1], torch.zeros(16, 8, device="cuda", dtype=t), torch.cat([Z, one], 1)[:1], act=act, k=k, bias=True)[2]
    assert torch.equal(torch.nan_to_num(both[:8], 99.0), torch.nan_to_num(slope, 99.0))
    n = len(values)
    assert all(torch.equal(torch.nan_to_num(r, 99.0), torch.nan_to_num(a[0], 99.0)) for a in (y, g) for r in a)
    return z.double(), y[0, :n].double(), g[0, :n].double(), both[8:8 + n].double(), slope[:n].double()


@pytest.mark.parametrize("dtype,rows,tile", ROUTES)
@pytest.mark.parametrize("k", (0.0, 0.2, 1.0, -0.5))
def test_relu_of_infinities(eng, tiled, dtype, rows, tile, k):
    """A LeakyReLU of slope 0 is a ReLU: 0 at -Inf.  Any other slope times -Inf is infinite; NaN stays."""
    inf, nan = float("inf"), float("nan")
    z, *values, slope = through_act(eng, tiled, dtype, rows, tile, "leakyRelu", k, [-inf, inf, nan, -2.0, 3.0, 0.0])
    want = torch.tensor([-inf * k if k else 0.0, inf, nan, -2.0 * k, 3.0, 0.0], device="cuda", dtype=torch.float64)
    for y in values:
        assert torch.equal(torch.isnan(y), torch.isnan(want))
        fine = ~torch.isnan(want)
        assert torch.equal(torch.isinf(y), torch.isinf(want)) and torch.equal(y[torch.isinf(want)], want[torch.isinf(want)])
        assert ((y - want)[fine & torch.isfinite(want)].abs() <= torch.finfo(TYPES[dtype]).eps * want[fine & torch.isfinite(want)].abs()).all()
    assert torch.equal(slope.to(TYPES[dtype]), torch.tensor([k, 1.0, k, k, 1.0, k], device="cuda").to(TYPES[dtype]).double().to(TYPES[dtype]))


@pytest.mark.parametrize("dtype,rows,tile", [r for r in ROUTES if r[0] != "f16"])
@pytest.mark.parametrize("act", ("silu", "gelu_tanh", "sigmoid"))
def test_small_values_of_large_arguments(eng, tiled, dtype, rows, tile, act):
    """Values far below zero, down to where fp32 has no normal numbers, in the forward pass and in the gradient of the ups alike.

    Errors: the exponential's 2 units of 2^-23 (of the type's fast one 2 + 1.16 |argument|), the argument's rounding as often as the argument is large - of
    gelu_tanh seven roundings of it -, three more roundings, and the output's; of denormals their spacing, times |z| where it is multiplied by it."""
    t = TYPES[dtype]
    half = torch.finfo(t).eps / 2
    values = {"gelu_tanh": [-9.0, -10.0, -10.1, -10.2, -10.25, -10.3], "silu": [-80.0, -87.0, -87.5, -88.0, -90.0, -92.0], "sigmoid": [-80.0, -86.0, -87.0, -87.3, -88.0, -100.0]}[act]
    z, y, g, up, _ = through_act(eng, tiled, dtype, rows, tile, act, 0.0, values)
    u = z if act != "gelu_tanh" else 1.5957691216057308 * (z + 0.044715 * z ** 3)
    s = torch.exp(u) / (1 + torch.exp(u))
    want = (s if act == "sigmoid" else z * s)[:len(values)]
    z, u = z[:len(values)], u[:len(values)]
    rel = 2.0 ** -23 * ((2 if dtype == "f32" else 2 + 1.16 * u.abs()) + 3) + (7 * 2.0 ** -24 * u.abs() if act == "gelu_tanh" else 0)
    tiny = (1 if act == "sigmoid" else z.abs()) * 2.0 ** -148 + (2.0 ** -134 if dtype == "bf16" else 2.0 ** -149)
    for got in (y, g, up):
        assert ((got - want).abs() <= (rel + half) * want.abs() * 1.01 + tiny).all(), (got, want)


# ---- what the rounding of deltaZ means in fp16 ----

@pytest.mark.parametrize("rows", (3, 200))
@pytest.mark.parametrize("tile", (0, 1))
def test_f16_deltaZ_has_the_range_of_f16(eng, tiled, rows, tile):
    """deltaY U of 90000 and of 1e-8 in fp16: Inf and 0 in the gradients of X and W; the bias gradient sums what they were before they were rounded."""
    tiled(tile)
    IC, OC, t = 64, 40, torch.float16
    gen = torch.Generator(device="cuda").manual_seed(8)
    X, W = torch.rand(rows, IC, device="cuda", generator=gen).add(1).to(t), torch.rand(2 * OC, IC, device="cuda", generator=gen).add(1).to(t)
    Z, dY = torch.ones(rows, 2 * OC, device="cuda", dtype=t), torch.ones(rows, OC, device="cuda", dtype=t)
    Z[1, OC + 3], dY[1, 3] = 300, 300                      # U and deltaY: deltaG is 90000
    Z[:, OC + 5], dY[:, 5] = 1e-4, 1e-4                    # deltaG is 1e-8 in every row, deltaU 1e-4
    dX, dW, dB = eng.fullConnect_glu_delta(dY, X, W, Z, act="none", bias=True)
    assert torch.isinf(dX[1]).all() and torch.isfinite(dX[0]).all() and torch.isfinite(dX[2:]).all()
    assert torch.isinf(dW[3]).all() and torch.isfinite(dW[4:]).all() and not dW[5].any()
    assert torch.isinf(dB[3])
    small = rows * float(Z[0, OC + 5]) * float(dY[0, 5])
    # (a sum of `rows` terms, rounded to fp16, whose denormals are 2^-24 apart)
    assert abs(float(dB[5]) - small) <= 2.0 ** -25 + rows * 2.0 ** -24 * small
