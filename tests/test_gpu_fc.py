"""FullConnect layers of a transformer (fullConnect, fullConnect_glu and their gradients) against 64-bit sums.

Bounds.  Products of 16-bit operands are exact in fp32; a tcgen05.mma adds 16 of them to an fp32 accumulator and truncates, so a sum of
K terms errs by at most (K / 16 + 8) 2^-22 of the sum of the terms' magnitudes (the 8: bias, partial sums of a split, residual); fp32
operands are multiplied as three bf16 planes, with at most 2^-23 of a product dropped and as many additions.  An activation's slope is at
most 1.13 in size and its evaluation errs by 2^-20 of value and sum.  An output is rounded once, eps / 2 of it; deltaZ is rounded before it is
multiplied, eps / 2 of each term.
"""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

K_SLOPE = 0.2
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ACTS = ("none", "leakyRelu", "sigmoid", "silu", "gelu", "gelu_tanh")


@pytest.fixture(scope="module")
def eng(pkg):
    return pkg.submodule("engine").Engine()


@pytest.fixture(scope="module")
def lib(pkg):
    return pkg.submodule("lib")


def act64(z, name, k=K_SLOPE):
    """Value and slope in float64, by autograd."""
    z = z.detach().clone().requires_grad_(True)
    y = {"none": lambda: z * 1.0, "leakyRelu": lambda: torch.where(z > 0, z, k * z), "sigmoid": lambda: torch.sigmoid(z), "silu": lambda: z * torch.sigmoid(z),
         "gelu": lambda: torch.nn.functional.gelu(z), "gelu_tanh": lambda: torch.nn.functional.gelu(z, approximate="tanh")}[name]()
    (d,) = torch.autograd.grad(y.sum(), z)
    return y.detach(), d


def rand(gen, *shape, scale=1.0, dtype=torch.float32):
    return torch.randn(shape, device="cuda", generator=gen).mul_(scale).to(dtype)


def sum_bound(K, S):
    return (K / 16 + 8) * 2.0 ** -22 * S


def check(name, got, ref, bound, dtype):
    half = torch.finfo(dtype).eps / 2
    assert got.dtype == dtype and tuple(got.shape) == tuple(ref.shape), (name, got.dtype, tuple(got.shape))
    err = (got.double() - ref).abs()
    limit = bound + half * (ref.abs() + bound) + torch.finfo(dtype).tiny * half
    bad = ~(err <= limit)
    assert not bad.any(), "%s: %d of %d outputs off, worst %.3g of its bound" % (name, int(bad.sum()), bad.numel(), float((err / limit).nan_to_num(1e9).max()))


def forward_case(eng, lib, dtype, rows, IC, OC, act, glu, bias, residual, save, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    t = TYPES[dtype]
    wide = 2 * OC if glu else OC
    X, W = rand(gen, rows, IC, dtype=t), rand(gen, wide, IC, scale=IC ** -0.5, dtype=t)
    B = rand(gen, wide, scale=0.5, dtype=t) if bias else None
    R = rand(gen, rows, OC, dtype=t) if residual else None
    out = eng.fullConnect_glu(X, W, B, act=act, k=K_SLOPE, save=save) if glu else eng.fullConnect(X, W, B, act=act, k=K_SLOPE, Residual=R, save=save)
    Y, Z = out if save else (out, None)
    z = X.double() @ W.double().T
    S = X.double().abs() @ W.double().abs().T
    if bias:
        z, S = z + B.double(), S + B.double().abs()
    ez = sum_bound(IC, S)
    if save:
        check("Z", Z, z, ez, t)
    g = z[:, :OC]
    v, _ = act64(g, act)
    ev = 1.13 * ez[:, :OC] + 2.0 ** -20 * (v.abs() + g.abs())
    if glu:
        u = z[:, OC:]
        ref, bound = v * u, ev * (u.abs() + ez[:, OC:]) + v.abs() * ez[:, OC:] + 2.0 ** -22 * (v * u).abs()
    else:
        ref, bound = v, ev
        if residual:
            ref = ref + R.double()
            bound = bound + 2.0 ** -22 * ref.abs()
    check("Y", Y, ref, bound, t)
    assert lib.device_status() == 0, lib.last_error()


# sizes from one row to several row tiles, reductions from one element to many blocks, widths that end inside every tile
SHAPES = [(1, 8, 8), (1, 4096, 1000), (2, 64, 24), (3, 1001, 77), (4, 2048, 520), (5, 96, 40), (17, 72, 264), (100, 640, 200), (128, 64, 128), (129, 1000, 260),
          (300, 333, 515), (513, 2048, 384), (1000, 24, 2056)]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("glu", (False, True), ids=("fc", "glu"))
def test_forward_shapes(eng, lib, dtype, glu, shape):
    rows, IC, OC = shape
    forward_case(eng, lib, dtype, rows, IC, OC, "silu" if glu else "gelu_tanh", glu, bias=True, residual=not glu, save=True)
    forward_case(eng, lib, dtype, rows, IC, OC, "gelu" if glu else "none", glu, bias=False, residual=False, save=False, seed=1)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("glu", (False, True), ids=("fc", "glu"))
@pytest.mark.parametrize("rows", (1, 3, 200))
def test_forward_activations(eng, lib, dtype, act, glu, rows):
    forward_case(eng, lib, dtype, rows, 256, 136, act, glu, bias=True, residual=not glu, save=True)


# CTA pairs, the plan by cost with deltaX and deltaW together or apart, tiles of some widths, tiles shared by 2, 4 and 8 CTAs
@pytest.mark.parametrize("tile", (1, 2, 3, 1016, 1064, 1112, 1256, 2080, 4048, 8256))
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("glu", (False, True), ids=("fc", "glu"))
@pytest.mark.parametrize("shape", [(1, 64, 8), (77, 200, 136), (700, 520, 1304), (2500, 128, 1544)], ids=lambda s: "x".join(map(str, s)))
def test_forward_tiles(eng, lib, dtype, glu, tile, shape):
    old = lib.set_option("FC_TILE", tile)
    try:
        rows, IC, OC = shape
        forward_case(eng, lib, dtype, rows, IC, OC, "silu", glu, bias=True, residual=not glu, save=True)
    finally:
        lib.set_option("FC_TILE", old)


def delta_case(eng, lib, dtype, rows, IC, OC, act, glu, bias, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    t = TYPES[dtype]
    half = torch.finfo(t).eps / 2
    wide = 2 * OC if glu else OC
    X, W, dY, Z = rand(gen, rows, IC, dtype=t), rand(gen, wide, IC, scale=IC ** -0.5, dtype=t), rand(gen, rows, OC, dtype=t), rand(gen, rows, wide, scale=2.0, dtype=t)
    held = Z.clone()
    fn = eng.fullConnect_glu_delta if glu else eng.fullConnect_delta
    dX, dW, dB = fn(dY, X, W, Z, act=act, k=K_SLOPE, bias=bias)
    assert torch.equal(Z, held)
    v, d = act64(Z.double()[:, :OC], act)
    y = dY.double()
    if glu:
        u = Z.double()[:, OC:]
        dZ = torch.cat([y * u * d, y * v], dim=1)
        eZ = 2.0 ** -20 * torch.cat([(y * u).abs() * (1 + d.abs() + Z.double()[:, :OC].abs()), y.abs() * (v.abs() + Z.double()[:, :OC].abs())], dim=1)
    else:
        dZ = y * d
        eZ = 2.0 ** -20 * y.abs() * (1 + d.abs() + Z.double().abs())
    if not glu and act == "none":
        eZ, rZ = torch.zeros_like(dZ), torch.zeros_like(dZ)
    else:
        rZ = (half if dtype != "f32" else 2.0 ** -24) * dZ.abs() + eZ
    a = dZ.abs() + rZ
    w, x = W.double().abs(), X.double().abs()
    check("deltaX", dX, dZ @ W.double(), rZ @ w + sum_bound(wide, a @ w), t)
    check("deltaW", dW, dZ.T @ X.double(), rZ.T @ x + sum_bound(rows, a.T @ x), t)
    if bias:
        check("deltaB", dB, dZ.sum(0), eZ.sum(0) + (rows + 16) * 2.0 ** -24 * a.sum(0), t)
    else:
        assert dB is None
    assert lib.device_status() == 0, lib.last_error()


@pytest.mark.parametrize("shape", [(1, 8, 8), (1, 640, 72), (5, 96, 40), (77, 333, 129), (130, 1000, 264), (513, 264, 1000), (2051, 136, 520)], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("glu", (False, True), ids=("fc", "glu"))
def test_delta_shapes(eng, lib, dtype, glu, shape):
    rows, IC, OC = shape
    delta_case(eng, lib, dtype, rows, IC, OC, "silu" if glu else "gelu", glu, bias=True)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("glu", (False, True), ids=("fc", "glu"))
def test_delta_activations(eng, lib, dtype, act, glu):
    delta_case(eng, lib, dtype, 150, 136, 200, act, glu, bias=act != "silu")


# CTA pairs, the plan by cost with deltaX and deltaW together or apart, tiles of some widths, tiles shared by 2, 4 and 8 CTAs
@pytest.mark.parametrize("tile", (1, 2, 3, 1016, 1064, 1112, 1256, 2080, 4048, 8256))
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(3, 8, 16), (700, 520, 1304), (1500, 1544, 200)], ids=lambda s: "x".join(map(str, s)))
def test_delta_tiles(eng, lib, dtype, tile, shape):
    old = lib.set_option("FC_TILE", tile)
    try:
        delta_case(eng, lib, dtype, *shape, "silu", True, bias=True)
    finally:
        lib.set_option("FC_TILE", old)


# ---- values ------------------------------------------------------------------------------------------------------

F32_FORMS = [(3, 0, "few rows"), (70, 2, "gathered"), (70, 1, "pairs")]


@pytest.mark.parametrize("rows,tile,_form", F32_FORMS, ids=[f[2] for f in F32_FORMS])
@pytest.mark.parametrize("glu", (False, True), ids=("fc", "glu"))
def test_f32_not_finite(eng, lib, rows, tile, _form, glu):
    """An Inf or NaN reaches the outputs that depend on it, as in 64 bits, and no other."""
    gen = torch.Generator(device="cuda").manual_seed(2)
    IC, OC = 200, 36
    X, W = rand(gen, rows, IC), rand(gen, (2 if glu else 1) * OC, IC)
    X[1, 7], X[2, 100], W[5, 150] = float("inf"), float("nan"), float("-inf")
    W[9, 7], X[0, 150] = 0.0, 0.0             # Inf * 0
    old = lib.set_option("FC_TILE", tile)
    try:
        Y, Z = eng.fullConnect_glu(X, W, act="leakyRelu", k=K_SLOPE, save=True) if glu else eng.fullConnect(X, W, act="none", save=True)
    finally:
        lib.set_option("FC_TILE", old)
    z = X.double() @ W.double().T
    assert torch.equal(torch.isnan(Z), torch.isnan(z)) and torch.equal(torch.isinf(Z), torch.isinf(z))
    assert torch.equal(Z[torch.isinf(z)].double(), z[torch.isinf(z)])
    fine = torch.isfinite(z)
    S = torch.where(torch.isfinite(X), X, 0).double().abs() @ torch.where(torch.isfinite(W), W, 0).double().abs().T
    assert ((Z.double() - z)[fine].abs() <= sum_bound(IC, S)[fine] + 2.0 ** -24 * z[fine].abs()).all()
    if glu:
        y = torch.where(z[:, :OC] > 0, z[:, :OC], K_SLOPE * z[:, :OC]) * z[:, OC:]
        assert torch.equal(torch.isnan(Y), torch.isnan(y)) and torch.equal(torch.isinf(Y), torch.isinf(y))
    assert lib.device_status() == 0


@pytest.mark.parametrize("rows,tile,_form", F32_FORMS, ids=[f[2] for f in F32_FORMS])
@pytest.mark.parametrize("x_scale,w_scale", [(1e-25, 1e-10), (1e-37, 1e11), (1e25, 1e10), (1e-38, 1.0)])
def test_f32_range(eng, lib, rows, tile, _form, x_scale, w_scale):
    """Operands and sums over the range of fp32, denormals (whose last place is an error of 2^-149 a term) among them."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    IC, OC = 130, 44
    X, W = rand(gen, rows, IC, scale=x_scale), rand(gen, OC, IC, scale=w_scale)
    old = lib.set_option("FC_TILE", tile)
    try:
        Y = eng.fullConnect(X, W)
        dX, dW, _ = eng.fullConnect_delta(torch.ones(rows, OC, device="cuda"), X, W)
    finally:
        lib.set_option("FC_TILE", old)
    for got, a, b in ((Y, X, W.T), (dX, torch.ones(rows, OC, device="cuda"), W), (dW, torch.ones(OC, rows, device="cuda"), X)):
        ref, S, K = a.double() @ b.double(), a.double().abs() @ b.double().abs(), a.shape[1]
        assert ((got.double() - ref).abs() <= sum_bound(K, S) + 2.0 ** -24 * ref.abs() + K * 2.0 ** -148).all()


@pytest.mark.parametrize("dtype", ("bf16", "f16"))
@pytest.mark.parametrize("rows,tile", [(2, 0), (12, 0), (70, 0), (70, 1), (70, 2016)])
def test_16bit_not_finite(eng, lib, dtype, rows, tile):
    gen = torch.Generator(device="cuda").manual_seed(4)
    t = TYPES[dtype]
    X, W = rand(gen, rows, 264, dtype=t), rand(gen, 80, 264, dtype=t)
    X[1, 7], W[5, 150], W[17, 3] = float("inf"), float("-inf"), float("nan")
    old = lib.set_option("FC_TILE", tile)
    try:
        Y = eng.fullConnect(X, W)
    finally:
        lib.set_option("FC_TILE", old)
    y = (X.double() @ W.double().T)
    assert torch.equal(torch.isnan(Y), torch.isnan(y)) and torch.equal(torch.isinf(Y), torch.isinf(y))


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", TYPES)
def test_activations_over_their_range(eng, dtype, act):
    """Values and slopes from the largest to the smallest arguments: X = z as one column, W = 1."""
    t = TYPES[dtype]
    top = min(float(torch.finfo(t).max), 1e30)
    m = torch.cat([torch.logspace(-8, 1.5, 400), torch.tensor([0.0, 60.0, 88.0, 90.0, 104.0, 200.0, 1e3, 1e4]), torch.tensor([min(1e15, top), top])]).cuda()
    z = torch.cat([m, -m]).to(t)
    X = torch.zeros(len(z), 8, device="cuda", dtype=t)
    X[:, 0] = z
    W = torch.zeros(8, 8, device="cuda", dtype=t)
    W[0, 0] = 1
    Y = eng.fullConnect(X, W, act=act, k=K_SLOPE)[:, 0]
    v, d = act64(z.double(), act)
    d = torch.where(torch.isfinite(d), d, (z > 0).double())          # (gelu of very large arguments: Inf * 0 in the derivative formula)
    half, tiny = torch.finfo(t).eps / 2, torch.finfo(t).tiny
    # exponentials of arguments beyond -87 underflow in fp32: what is left of the value is below 1e-35
    assert ((Y.double() - v).abs() <= half * v.abs() + 2.0 ** -19 * v.abs() + 2.0 ** -24 * torch.minimum(z.double().abs(), torch.tensor(1.0).cuda()) + 1e-35 + tiny * half).all()
    dY = torch.zeros(len(z), 8, device="cuda", dtype=t)
    dY[:, 0] = 1
    Z = torch.zeros(len(z), 8, device="cuda", dtype=t)
    Z[:, 0] = z
    I = torch.eye(8, device="cuda", dtype=t)
    dX, _, _ = eng.fullConnect_delta(dY, X, I, Z, act=act, k=K_SLOPE)
    # (slopes pass through zero: 2^-19 of the terms they are the sum of)
    assert ((dX[:, 0].double() - d).abs() <= 2 * half * d.abs() + 2.0 ** -19 * (d.abs() + v.abs().clamp(max=1.0) + 2.0 ** -4) + tiny * half).all()


def test_gradients_against_differences(eng):
    """d/dh of sum(C * Y) along random directions, by central differences of the definition in 64 bits."""
    gen = torch.Generator(device="cuda").manual_seed(6)
    rows, IC, OC, h = 9, 20, 12, 1e-5
    for glu in (False, True):
        for act in ACTS:
            wide = 2 * OC if glu else OC
            X, W, B, C = rand(gen, rows, IC), rand(gen, wide, IC, scale=0.3), rand(gen, wide), rand(gen, rows, OC)

            def loss(x, w, b):
                z = x @ w.T + b
                v = act64(z[:, :OC], act)[0]
                return float((C.double() * (v * z[:, OC:] if glu else v)).sum())

            fn, gr = (eng.fullConnect_glu, eng.fullConnect_glu_delta) if glu else (eng.fullConnect, eng.fullConnect_delta)
            _, Z = fn(X, W, B, act=act, k=K_SLOPE, save=True)
            grads = gr(C, X, W, Z, act=act, k=K_SLOPE, bias=True)
            at = [t.double() for t in (X, W, B)]
            for i, g in enumerate(grads):
                v = torch.randn(at[i].shape, device="cuda", generator=gen, dtype=torch.float64)
                up, down = list(at), list(at)
                up[i], down[i] = at[i] + h * v, at[i] - h * v
                want = (loss(*up) - loss(*down)) / (2 * h)
                got = float((g.double() * v).sum())
                # differences err by h^2 and by rounding of the loss / h; the gradients by fp32 sums of up to 200 terms
                assert abs(got - want) <= 1e-4 * float((g.double() * v).abs().sum()) + 1e-5, (glu, act, i)


# ---- calls -------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
def test_leading_dimensions_views_and_empty_batches(eng, dtype):
    gen = torch.Generator(device="cuda").manual_seed(7)
    t = TYPES[dtype]
    W, B = rand(gen, 48, 72, scale=0.1, dtype=t), rand(gen, 48, dtype=t)
    X = rand(gen, 5, 7, 72, dtype=t)
    want, wz = eng.fullConnect(X.reshape(35, 72), W, B, act="silu", save=True)
    Y, Z = eng.fullConnect(X, W, B, act="silu", save=True)
    assert Y.shape == (5, 7, 48) and Z.shape == (5, 7, 48) and torch.equal(Y.reshape(35, 48), want) and torch.equal(Z.reshape(35, 48), wz)
    assert torch.equal(eng.fullConnect(X[2, 3], W, B, act="silu"), eng.fullConnect(X[2, 3].reshape(1, 72), W, B, act="silu").reshape(48))
    # transposed, offset and strided views
    flat = rand(gen, 35 * 72 + 1, dtype=t)
    shifted = flat[1:].reshape(35, 72)
    assert torch.equal(eng.fullConnect(shifted, W), eng.fullConnect(shifted.clone(), W))
    assert torch.equal(eng.fullConnect(X[:, ::2], W), eng.fullConnect(X[:, ::2].contiguous(), W))
    Wt = W.T.contiguous().T
    assert not Wt.is_contiguous() and torch.equal(eng.fullConnect(X, Wt), eng.fullConnect(X, W))
    dY = rand(gen, 5, 7, 48, dtype=t)
    whole = eng.fullConnect_delta(dY, X, W, Z, act="silu", bias=True)
    assert whole[0].shape == X.shape and whole[1].shape == W.shape and whole[2].shape == B.shape
    again = eng.fullConnect_delta(dY.transpose(0, 1).contiguous().transpose(0, 1), X, Wt, Z, act="silu", bias=True)
    assert all(torch.equal(a, b) for a, b in zip(whole, again))
    # nothing in, nothing out
    none = X[:0]
    for glu in (False, True):
        fn, gr = (eng.fullConnect_glu, eng.fullConnect_glu_delta) if glu else (eng.fullConnect, eng.fullConnect_delta)
        y, z = fn(none, W, B, save=True)
        assert y.shape == (0, 7, 24 if glu else 48) and z.shape == (0, 7, 48)
        dx, dw, db = gr(y, none, W, z, act="silu", bias=True)
        assert dx.shape == none.shape and dw.shape == W.shape and not dw.any() and db.shape == (48,) and not db.any()


def test_lazily_negated_views(eng):
    c = torch.randn(12, 16, device="cuda", dtype=torch.complex64)
    X = c.conj().imag
    W = torch.randn(8, 16, device="cuda")
    assert X.is_neg()
    ref = X.double() @ W.double().T
    assert (eng.fullConnect(X, W).double() - ref).abs().max() < 1e-5


@pytest.mark.parametrize("dtype,rows", [("f32", 3), ("f32", 300), ("bf16", 3), ("bf16", 12), ("bf16", 300), ("bf16", 3000), ("f16", 40)])
def test_in_place_residual_and_delta(eng, lib, dtype, rows):
    """Y may be the residual's memory, deltaZ that of Z."""
    import ctypes as C
    gen = torch.Generator(device="cuda").manual_seed(8)
    t = TYPES[dtype]
    code = {"f32": 0, "bf16": 1, "f16": 2}[dtype]
    IC, OC = 520, 264
    X, W, R = rand(gen, rows, IC, dtype=t), rand(gen, OC, IC, scale=0.05, dtype=t), rand(gen, rows, OC, dtype=t)
    want = eng.fullConnect(X, W, Residual=R)
    eng.base.fullConnect(R, X, W, rows, IC, OC, code, 0, 0.0, None, R, None)
    assert torch.equal(R, want)
    W2, dY, Z = rand(gen, 2 * OC, IC, scale=0.05, dtype=t), rand(gen, rows, OC, dtype=t), rand(gen, rows, 2 * OC, dtype=t)
    want = eng.fullConnect_glu_delta(dY, X, W2, Z)
    dX, dW = torch.empty_like(X), torch.empty_like(W2)
    eng.base.fullConnect_delta(dX, dW, None, dY, X, W2, Z, Z, rows, IC, OC, code, lib.ACTS["silu"], 0.0, True)
    assert torch.equal(dX, want[0]) and torch.equal(dW, want[1])


@pytest.mark.parametrize("dtype", TYPES)
def test_some_gradients_only(eng, lib, dtype):
    gen = torch.Generator(device="cuda").manual_seed(9)
    t = TYPES[dtype]
    code = {"f32": 0, "bf16": 1, "f16": 2}[dtype]
    rows, IC, OC = 257, 136, 72
    X, W, dY, Z = rand(gen, rows, IC, dtype=t), rand(gen, OC, IC, dtype=t), rand(gen, rows, OC, dtype=t), rand(gen, rows, OC, dtype=t)
    want = eng.fullConnect_delta(dY, X, W, Z, act="gelu", bias=True)
    for keep in ((0,), (1,), (2,), (0, 2), (1, 2)):
        out = [torch.empty_like(w) if i in keep else None for i, w in enumerate(want)]
        dZ = torch.empty_like(Z)
        eng.base.fullConnect_delta(out[0], out[1], out[2], dY, X if 1 in keep else None, W if 0 in keep else None, Z, dZ, rows, IC, OC, code, lib.ACTS["gelu"], 0.0)
        for i in keep:
            if dtype == "f32":          # (kernels are chosen by what is asked for together)
                assert (out[i] - want[i]).abs().max() <= 1e-4
            else:
                assert torch.equal(out[i], want[i])


def test_rows_behind_the_last_stay(eng, lib):
    """Outputs end at the last row and column: a box, a word or a tile that passes them writes nothing there."""
    gen = torch.Generator(device="cuda").manual_seed(10)
    for dtype, code in (("f32", 0), ("bf16", 1), ("f16", 2)):
        t = TYPES[dtype]
        for rows in (1, 5, 13, 70, 200):
            for tile in (0, 1, 2, 1048, 2112):
                IC, OC = 72, 40
                X, W = rand(gen, rows, IC, dtype=t), rand(gen, OC, IC, dtype=t)
                n = rows * OC
                Y = torch.full((n + 4096,), 7.0, device="cuda").to(t)
                Z = torch.full((n + 4096,), 7.0, device="cuda").to(t)
                old = lib.set_option("FC_TILE", tile)
                try:
                    eng.base.fullConnect(Y, X, W, rows, IC, OC, code, lib.ACTS["silu"], 0.0, None, None, Z)
                finally:
                    lib.set_option("FC_TILE", old)
                assert (Y[n:] == 7).all() and (Z[n:] == 7).all(), (dtype, rows, tile)


@pytest.mark.parametrize("dtype,rows", [("f32", 2), ("f32", 600), ("bf16", 2), ("bf16", 600), ("bf16", 2048)])
def test_capture_and_replay(eng, lib, dtype, rows):
    gen = torch.Generator(device="cuda").manual_seed(11)
    t = TYPES[dtype]
    IC, OC = 1024, 520
    X, W, dY = rand(gen, rows, IC, dtype=t), rand(gen, 2 * OC, IC, scale=0.03, dtype=t), rand(gen, rows, OC, dtype=t)

    def step():
        Y, Z = eng.fullConnect_glu(X, W, save=True)
        return (Y,) + eng.fullConnect_glu_delta(dY, X, W, Z, bias=True)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()                        # (once eagerly: the stream's scratch)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            out = step()
    X.copy_(rand(gen, rows, IC, dtype=t))
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        g.replay()
        want = step()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, want))
    del g
    # a stream that has no scratch yet: partial column sums need some, the rest runs without
    lib.release_workspace()
    s = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        Y, Z = eng.fullConnect_glu(X, W, save=True)
        dX, dW, _ = eng.fullConnect_glu_delta(dY, X, W, Z)
        with pytest.raises(lib.AlphaConvError) as e:
            eng.fullConnect_glu_delta(dY, X, W, Z, bias=True)
        assert e.value.code == -6
    g.replay()
    torch.cuda.synchronize()
    assert (Y.double() - want[0].double()).abs().max() <= 0.02 * want[0].double().abs().max()
    assert (dW.double() - want[2].double()).abs().max() <= 0.02 * want[2].double().abs().max()
    assert (dX.double() - want[1].double()).abs().max() <= 0.02 * want[1].double().abs().max()


def test_own_stream_and_two_at_once(pkg):
    """Engines with streams of their own, working at the same time on odd sizes (padded copies in each call)."""
    engine = pkg.submodule("engine")
    gen = torch.Generator(device="cuda").manual_seed(12)
    streams = [torch.cuda.Stream() for _ in range(2)]
    engs = [engine.Engine(engine.CudaFloat32EngineBase(stream=s)) for s in streams]
    X, W, dY = rand(gen, 301, 333), rand(gen, 2 * 129, 333, scale=0.05), rand(gen, 301, 129)
    one = engine.Engine()
    Y, Z = one.fullConnect_glu(X, W, save=True)
    want = (Y, Z) + one.fullConnect_glu_delta(dY, X, W, Z, bias=True)
    torch.cuda.synchronize()
    got = []
    for _ in range(10):
        for e in engs:
            y, z = e.fullConnect_glu(X, W, save=True)
            got.append((y, z) + e.fullConnect_glu_delta(dY, X, W, z, bias=True))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for out in got for a, b in zip(out, want))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("glu", (False, True), ids=("fc", "glu"))
@pytest.mark.parametrize("rows", (2, 300))
def test_workspace_bytes_are_enough(eng, lib, dtype, glu, rows):
    gen = torch.Generator(device="cuda").manual_seed(13)
    t = TYPES[dtype]
    code = {"f32": 0, "bf16": 1, "f16": 2}[dtype]
    IC, OC = 2048, 512
    wide = 2 * OC if glu else OC
    X, W, dY, Z = rand(gen, rows, IC, dtype=t), rand(gen, wide, IC, dtype=t), rand(gen, rows, OC, dtype=t), rand(gen, rows, wide, dtype=t)
    shape = lib.AlphaFcShape(rows, IC, OC, code, lib.ACTS["silu"], 0.0)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    for tile in (0, 1, 2):
        old = lib.set_option("FC_TILE", tile)
        try:
            need = {op: lib.fullConnect_workspace_bytes(shape, glu, op) for op in ("forward", "deltaX")}
            with torch.cuda.stream(s):
                for op, n in need.items():
                    block = torch.empty(max(n, 256), dtype=torch.uint8, device="cuda")
                    lib.set_workspace(s.cuda_stream, block.data_ptr(), n)
                    before = lib.workspace_in_use()
                    if op == "forward":
                        fn = eng.fullConnect_glu if glu else eng.fullConnect
                        fn(X, W, act="silu")
                    else:
                        (eng.fullConnect_glu_delta if glu else eng.fullConnect_delta)(dY, X, W, Z, act="silu", bias=True)
                    assert lib.workspace_in_use() == before
                    torch.cuda.synchronize()
        finally:
            lib.set_workspace(s.cuda_stream, None, 0)
            lib.set_option("FC_TILE", old)


def test_same_bits(eng):
    gen = torch.Generator(device="cuda").manual_seed(14)
    for dtype in TYPES:
        t = TYPES[dtype]
        for rows, IC, OC in ((1, 4096, 2048), (16, 4096, 520), (100, 4096, 264), (700, 2048, 1032)):
            X, W, dY = rand(gen, rows, IC, dtype=t), rand(gen, 2 * OC, IC, scale=0.02, dtype=t), rand(gen, rows, OC, dtype=t)

            def step():
                Y, Z = eng.fullConnect_glu(X, W, save=True)
                return (Y, Z) + eng.fullConnect_glu_delta(dY, X, W, Z, bias=True)
            first = step()
            for _ in range(5):
                assert all(torch.equal(a, b) for a, b in zip(first, step()))


@pytest.mark.parametrize("sms", (1, 2, 7, 100))
def test_sm_budget(eng, lib, sms):
    old = lib.set_option("SM_BUDGET", sms)
    try:
        for dtype in TYPES:
            for tile in (0, 1, 2048):
                o = lib.set_option("FC_TILE", tile)
                try:
                    forward_case(eng, lib, dtype, 300, 264, 520, "silu", True, True, False, True)
                    delta_case(eng, lib, dtype, 300, 264, 520, "silu", True, True)
                finally:
                    lib.set_option("FC_TILE", o)
    finally:
        lib.set_option("SM_BUDGET", old)


def test_more_than_2_31_elements(eng):
    """A 16-bit Z of 2.3 billion elements, read and written beyond 32-bit offsets."""
    gen = torch.Generator(device="cuda").manual_seed(15)
    rows, IC, OC = 70000, 64, 16384
    X, W = rand(gen, rows, IC, dtype=torch.bfloat16), rand(gen, 2 * OC, IC, scale=0.125, dtype=torch.bfloat16)
    Y, Z = eng.fullConnect_glu(X, W, save=True)
    some = torch.tensor([0, 1, 32767, 32768, 65535, 65536, 69998, 69999], device="cuda")
    z = X[some].double() @ W.double().T
    assert ((Z[some].double() - z).abs() <= 2.0 ** -8 * z.abs() + 1e-4).all()
    v = z[:, :OC] * torch.sigmoid(z[:, :OC]) * z[:, OC:]
    assert ((Y[some].double() - v).abs() <= 2.0 ** -8 * v.abs() + 1e-3).all()
    dY = torch.zeros_like(Y)
    dY[some] = 1
    dX, dW, dB = eng.fullConnect_glu_delta(dY, X, W, Z, bias=True)
    s, d = act64(Z[some].double()[:, :OC], "silu")
    dZ = torch.cat([Z[some].double()[:, OC:] * d, s], dim=1)
    ref = dZ @ W.double()
    S = dZ.abs() @ W.double().abs()
    assert ((dX[some].double() - ref).abs() <= 2.0 ** -8 * (ref.abs() + S) + sum_bound(2 * OC, S)).all()
    rest = torch.ones(rows, dtype=torch.bool, device="cuda")
    rest[some] = False
    assert not dX[rest].any()
    assert ((dB.double() - dZ.sum(0)).abs() <= 2.0 ** -8 * dZ.sum(0).abs() + 1e-5 * (1 + dZ.abs().sum(0))).all()


# ---- the operators together ---------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,tol", [("f32", 2e-5), ("bf16", 2e-2), ("f16", 3e-3)])
@pytest.mark.parametrize("tokens", [(1, 1), (2, 77)])
def test_feed_forward_step(eng, dtype, tol, tokens):
    """A transformer's feed-forward layer, trained for one step: gated block, projection with residual, all gradients, clipped.  Against
    autograd in 64 bits; errors (2-norm) are those of a few roundings of eps / 2 each, fp32 sums for f32."""
    gen = torch.Generator(device="cuda").manual_seed(16)
    t = TYPES[dtype]
    D, H = 256, 700
    X, W1, W2, B2 = rand(gen, *tokens, D, dtype=t), rand(gen, 2 * H, D, scale=D ** -0.5, dtype=t), rand(gen, D, H, scale=H ** -0.5, dtype=t), rand(gen, D, dtype=t)
    dY = rand(gen, *tokens, D, dtype=t)
    A, Z = eng.fullConnect_glu(X, W1, save=True)
    Y = eng.fullConnect(A, W2, B2, Residual=X)
    dA, dW2, dB2 = eng.fullConnect_delta(dY, A, W2, bias=True)
    dX, dW1, _ = eng.fullConnect_glu_delta(dA, X, W1, Z)
    dX = dX + dY
    master = [torch.empty_like(g, dtype=torch.float32) for g in (dW1, dW2, dB2)]
    norm = eng.clip_grad_norm([g.contiguous() for g in (dW1, dW2, dB2)], 0.5, Out=master)

    x, w1, w2, b2 = [v.double().requires_grad_(True) for v in (X, W1, W2, B2)]
    z = x @ w1.T
    y = (z[..., :H] * torch.sigmoid(z[..., :H]) * z[..., H:]) @ w2.T + b2 + x
    grads = torch.autograd.grad((y * dY.double()).sum(), (x, w1, w2, b2))
    rel = lambda a, b: float((a.double() - b).norm() / b.norm())
    assert rel(Y, y.detach()) <= tol
    for got, want in zip((dX, dW1, dW2, dB2), grads):
        assert rel(got, want) <= tol
    n = torch.sqrt(sum((g ** 2).sum() for g in grads[1:]))
    assert abs(float(norm) - float(n)) <= tol * float(n)
    for m, g in zip(master, grads[1:]):
        assert rel(m, g * min(1.0, 0.5 / (float(n) + 1e-6))) <= 2 * tol


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("glu", (False, True), ids=("fc", "glu"))
@pytest.mark.parametrize("tile", (0, 1, 2, 2064))
def test_what_padding_columns_hold_does_not_matter(eng, lib, dtype, glu, tile):
    """OC = 44 in tensors of 48 columns, the last four of every input NaN."""
    gen = torch.Generator(device="cuda").manual_seed(17)
    t = TYPES[dtype]
    code = {"f32": 0, "bf16": 1, "f16": 2}[dtype]
    IC, OC, P, H = 136, 44, 48, 2 if glu else 1
    old = lib.set_option("FC_TILE", tile)
    try:
        for rows in (1, 9, 70, 300):
            X, W, B = rand(gen, rows, IC, dtype=t), rand(gen, H * OC, IC, scale=0.1, dtype=t), rand(gen, H * OC, dtype=t)
            R, dY = rand(gen, rows, OC, dtype=t), rand(gen, rows, OC, dtype=t)

            def wide(a, n):                      # (..., n * OC) as (..., n, P) with NaN behind
                out = torch.full(a.shape[:-1] + (n, P), float("nan"), dtype=t, device="cuda")
                out[..., :OC] = a.reshape(a.shape[:-1] + (n, OC))
                return out
            for act in ("silu",) if glu else ("silu", "none"):
                if glu:
                    want, wz = eng.fullConnect_glu(X, W, B, act=act, save=True)
                else:
                    want, wz = eng.fullConnect(X, W, B, act=act, Residual=R, save=True)
                Y, Z = torch.empty(rows, P, dtype=t, device="cuda"), torch.empty(rows, H, P, dtype=t, device="cuda")
                if glu:
                    eng.base.fullConnect_glu(Y, X, W, rows, IC, OC, code, lib.ACTS[act], 0.0, wide(B, 2), Z)
                else:
                    eng.base.fullConnect(Y, X, W, rows, IC, OC, code, lib.ACTS[act], 0.0, wide(B, 1), wide(R, 1), Z)
                assert torch.equal(Y[:, :OC], want) and torch.equal(Z[..., :OC].reshape(rows, H * OC), wz)
                grads = (eng.fullConnect_glu_delta if glu else eng.fullConnect_delta)(dY, X, W, wz, act=act, bias=True)
                dX, dW, dB = torch.empty_like(X), torch.empty_like(W), torch.empty(H, P, dtype=t, device="cuda")
                eng.base.fullConnect_delta(dX, dW, dB, wide(dY, 1), X, W, wide(wz, H), torch.empty_like(Z), rows, IC, OC, code, lib.ACTS[act], 0.0, glu)
                for got, ref in ((dX, grads[0]), (dW, grads[1]), (dB[:, :OC].reshape(-1), grads[2])):
                    # (fp32: where the padding makes a sum NaN it is formed once more by FMAs)
                    assert torch.equal(got, ref) if dtype != "f32" else (got - ref).abs().max() <= 1e-5 * ref.abs().max()
    finally:
        lib.set_option("FC_TILE", old)
    assert lib.device_status() == 0


@pytest.mark.parametrize("rows,IC,OC", [(608, 536, 745), (1005, 560, 1488), (658, 144, 723), (1044, 664, 358), (128, 72, 40), (4169, 936, 1422)])
@pytest.mark.parametrize("glu", (False, True), ids=("fc", "glu"))
@pytest.mark.parametrize("dtype", ("bf16", "f16"))
def test_both_gradients_by_one_launch(eng, lib, dtype, glu, rows, IC, OC):
    """deltaX and deltaW in one launch have the bits of a launch each of the same tiles, and the same sums in any case."""
    delta_case(eng, lib, dtype, rows, IC, OC, "silu", glu, True)
    gen = torch.Generator(device="cuda").manual_seed(18)
    t = TYPES[dtype]
    H = 2 if glu else 1
    X, W, dY, Z = rand(gen, rows, IC, dtype=t), rand(gen, H * OC, IC, scale=0.1, dtype=t), rand(gen, rows, OC, dtype=t), rand(gen, rows, H * OC, dtype=t)
    fn = eng.fullConnect_glu_delta if glu else eng.fullConnect_delta
    both = fn(dY, X, W, Z, act="silu")
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(both[:2], fn(dY, X, W, Z, act="silu")[:2]))
    old = lib.set_option("FC_TILE", 3)
    try:
        apart = fn(dY, X, W, Z, act="silu")
    finally:
        lib.set_option("FC_TILE", old)
    for a, b in zip(both[:2], apart[:2]):
        # (a reduction split in another way differs in the last place)
        assert ((a.double() - b.double()).abs() <= torch.finfo(t).eps * b.double().abs() + 2e-3 * torch.finfo(t).eps / 2.0 ** -7 * b.double().abs().max()).all()


@pytest.mark.parametrize("shape", [(1, 64, 8), (77, 200, 136), (257, 132, 129), (700, 520, 1304), (2500, 128, 1544), (1500, 1544, 200)], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("glu", (False, True), ids=("fc", "glu"))
def test_f32_pairs_of_128_columns(eng, lib, glu, shape):
    """The pair kernel's narrow tiles, parts of a reduction included: forward and gradients, finite or not."""
    rows, IC, OC = shape
    old = lib.set_option("FC_TILE", 11)
    try:
        forward_case(eng, lib, "f32", rows, IC, OC, "gelu", glu, bias=True, residual=not glu, save=True)
        assert "256x128" in lib.last_plan(), lib.last_plan()
        delta_case(eng, lib, "f32", rows, IC, OC, "silu", glu, True)
        assert "256x128" in lib.last_plan(), lib.last_plan()
    finally:
        lib.set_option("FC_TILE", old)
    test_f32_not_finite(eng, lib, 70, 11, "pairs of 128 columns", glu)


@pytest.mark.parametrize("x_scale,w_scale", [(1e-25, 1e-10), (1e-37, 1e11), (1e25, 1e10), (1e-38, 1.0)])
def test_f32_range_of_128_columns(eng, lib, x_scale, w_scale):
    test_f32_range(eng, lib, 70, 11, "pairs of 128 columns", x_scale, w_scale)


@pytest.mark.parametrize("shape", [(1, 64, 8), (77, 200, 136), (257, 136, 129), (700, 520, 1304), (2500, 128, 1544), (1500, 1544, 200)], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("dtype", ("bf16", "f16"))
@pytest.mark.parametrize("glu", (False, True), ids=("fc", "glu"))
def test_16bit_pairs_of_128_columns(eng, lib, dtype, glu, shape):
    rows, IC, OC = shape
    old = lib.set_option("FC_TILE", 11)
    try:
        forward_case(eng, lib, dtype, rows, IC, OC, "silu", glu, bias=True, residual=not glu, save=True)
        assert "pair 256x128" in lib.last_plan(), lib.last_plan()
        delta_case(eng, lib, dtype, rows, IC, OC, "gelu", glu, True)
        assert "pair 256x128" in lib.last_plan(), lib.last_plan()
    finally:
        lib.set_option("FC_TILE", old)
