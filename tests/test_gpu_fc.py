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


# CTA pairs, the plan by cost, tiles of some widths, tiles shared by 2, 4 and 8 CTAs
@pytest.mark.parametrize("tile", (1, 2, 1016, 1064, 1112, 1256, 2080, 4048, 8256))
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


# CTA pairs, the plan by cost, tiles of some widths, tiles shared by 2, 4 and 8 CTAs
@pytest.mark.parametrize("tile", (1, 2, 1016, 1064, 1112, 1256, 2080, 4048, 8256))
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(3, 8, 16), (700, 520, 1304), (1500, 1544, 200)], ids=lambda s: "x".join(map(str, s)))
def test_delta_tiles(eng, lib, dtype, tile, shape):
    old = lib.set_option("FC_TILE", tile)
    try:
        delta_case(eng, lib, dtype, *shape, "silu", True, bias=True)
    finally:
        lib.set_option("FC_TILE", old)
