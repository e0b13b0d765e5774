"""groupNorm and groupNorm_delta against 64-bit results.

Bounds, per element, with e = 2^-24 and u = eps / 2 of the type.  A mean of n numbers errs by at most 24 e max|x| here (trees of fewer than 24 levels of additions, however they
are cut), so that z = (x - mean) rstd gamma + beta errs by |gamma| rstd 24 e max|x| and 64 e (|xh gamma| + |beta|) for rstd, the products and the sum.  An activation passes an error
on with its slope, at most 1.13, and errs itself by 2^-20 of its value in fp32 and 2^-16 in 16 bits (the fitted distribution function).  The output is rounded once.
Gradients: dz errs by |dy| times the slope's error (1.2 of z's, and 2^-16 or 2^-20 of 1 + |z|); a sum errs by the sum of its terms' errors and 64 e of the sum of their magnitudes."""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ACTS = ("none", "leakyRelu", "sigmoid", "silu", "gelu", "gelu_tanh")
K, E = 0.2, 2.0 ** -24


@pytest.fixture(scope="module")
def eng(pkg):
    return pkg.submodule("engine").Engine()


@pytest.fixture(scope="module")
def lib(pkg):
    return pkg.submodule("lib")


def act64(z, name):
    if name == "none":
        return z
    if name == "leakyRelu":
        return torch.where(z > 0, z, K * z)
    if name == "sigmoid":
        return torch.sigmoid(z)
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "gelu":
        return 0.5 * z * torch.erfc(-z / 2 ** 0.5)
    return 0.5 * z * (1 + torch.tanh((2 / torch.pi) ** 0.5 * (z + 0.044715 * z ** 3)))


def reference(X, G, gamma, beta, eps, act, dY=None, mean=None, rstd=None):
    """Y, mean, rstd, z in 64 bits; with dY the gradients by differentiation, mean and rstd being functions of X."""
    x = X.double().requires_grad_(dY is not None)
    N, C = X.shape[0], X.shape[-1]
    ga = torch.ones(C, dtype=torch.float64, device=X.device) if gamma is None else gamma.double()
    be = torch.zeros(C, dtype=torch.float64, device=X.device) if beta is None else beta.double()
    ga.requires_grad_(dY is not None)
    be.requires_grad_(dY is not None)
    t = x.reshape(N, -1, G, C // G)
    m = t.mean((1, 3), keepdim=True)
    r = ((t - m).square().mean((1, 3), keepdim=True) + eps) ** -0.5
    xh = ((t - m) * r).reshape(X.shape)
    z = xh * ga + be
    y = act64(z, act)
    if dY is None:
        return y, m.reshape(N, G), r.reshape(N, G), z, xh
    return torch.autograd.grad(y, (x, ga, be), dY.double())


def make(shape, dtype, seed=0, affine="same", offset=0.0, spread=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    C, t = shape[-1], TYPES[dtype]
    X = (torch.randn(shape, device="cuda", generator=g) * spread + offset + torch.randn(C, device="cuda", generator=g) * 0.5).to(t)
    a = torch.float32 if affine == "f32" else t
    gamma, beta = (None, None) if affine == "none" else ((1 + 0.3 * torch.randn(C, device="cuda", generator=g)).to(a), (0.3 * torch.randn(C, device="cuda", generator=g)).to(a))
    return X, torch.randn(shape, device="cuda", generator=g).to(t), gamma, beta


def per_channel(v, shape, G):
    """[N, G] values spread over a tensor's elements."""
    C = shape[-1]
    return v.repeat_interleave(C // G, 1).reshape((shape[0],) + (1,) * (len(shape) - 2) + (C,))


def check_forward(eng, X, G, gamma, beta, act, eps=1e-5):
    Y, mean, rstd = eng.groupNorm(X, G, gamma, beta, eps=eps, act=act, k=K, save=True)
    y, m, r, z, xh = reference(X, G, gamma, beta, eps, act)
    big = X.double().abs().amax(tuple(range(1, X.dim())))[:, None]
    assert Y.dtype == X.dtype and Y.shape == X.shape and mean.dtype == torch.float32
    assert ((mean.double() - m).abs() <= 26 * E * big).all()
    # a variance errs by 64 e of itself and the square of the mean's error; half as much of a root
    assert ((rstd.double() - r).abs() <= r * (64 * E + 0.5 * r * r * (26 * E * big) ** 2)).all()
    ga = 1.0 if gamma is None else gamma.double().abs()
    be = 0.0 if beta is None else beta.double().abs()
    zerr = ga * per_channel(r * 26 * E * big, X.shape, G) + 64 * E * ((xh * ga).abs() + be)
    own = 2.0 ** (-20 if X.dtype == torch.float32 else -16)
    limit = 1.13 * zerr + (own + torch.finfo(X.dtype).eps / 2) * y.abs() + own * 1e-3 * (act != "none") + torch.finfo(X.dtype).smallest_normal
    assert ((Y.double() - y).abs() <= limit).all(), float(((Y.double() - y).abs() / limit).max())
    assert torch.equal(Y, eng.groupNorm(X, G, gamma, beta, eps=eps, act=act, k=K))
    return mean, rstd


def check_delta(eng, X, dY, G, gamma, beta, act, mean, rstd, eps=1e-5):
    dX, dG, dB = eng.groupNorm_delta(dY, X, mean, rstd, gamma, beta, act=act, k=K)
    rx, rg, rb = reference(X, G, gamma, beta, eps, act, dY)
    _, m, r, z, xh = reference(X, G, gamma, beta, eps, act)
    own = 2.0 ** (-20 if X.dtype == torch.float32 else -16)
    ga = torch.ones((), dtype=torch.float64, device=X.device) if gamma is None else gamma.double().abs()
    be = 0.0 if beta is None else beta.double().abs()
    big = X.double().abs().amax(tuple(range(1, X.dim())))[:, None]
    xerr = per_channel(r * 26 * E * big, X.shape, G) + 64 * E * xh.abs()
    zerr = ga * xerr + 64 * E * be
    dz = dY.double().abs() * 1.13
    dzerr = dY.double().abs() * (1.2 * zerr + own * (1 + z.abs())) + 4 * E * dz
    if act == "leakyRelu":               # the slope jumps at 0: an element whose z may be of either sign
        dzerr = dzerr + dY.double().abs() * (z.abs() <= zerr)
    lead = tuple(range(X.dim() - 1))
    half = torch.finfo(X.dtype).eps / 2
    tiny = torch.finfo(X.dtype).smallest_normal
    if gamma is not None:
        ha = torch.finfo(gamma.dtype).eps / 2
        lg = (dzerr * xh.abs() + dz * xerr + 64 * E * dz * xh.abs()).sum(lead) + ha * rg.abs() + tiny
        lb = (dzerr + 64 * E * dz).sum(lead) + ha * rb.abs() + tiny
        assert dG.dtype == gamma.dtype and ((dG.double() - rg).abs() <= lg).all(), float(((dG.double() - rg).abs() / lg).max())
        assert ((dB.double() - rb).abs() <= lb).all(), float(((dB.double() - rb).abs() / lb).max())
    else:
        assert dG is None and dB is None
    N, C = X.shape[0], X.shape[-1]
    group = lambda t: per_channel(t.reshape(N, -1, G, C // G).mean((1, 3)), X.shape, G)       # noqa: E731
    e1, s1 = group((dzerr + 64 * E * dz) * ga), group(dz * ga)
    e2, s2 = group((dzerr * xh.abs() + dz * xerr + 64 * E * dz * xh.abs()) * ga), group(dz * ga * xh.abs())
    R = per_channel(r, X.shape, G)
    limit = R * (dzerr * ga + e1 + xh.abs() * e2 + xerr * s2 + 96 * E * (dz * ga + s1 + xh.abs() * s2)) + half * rx.abs() + tiny
    assert dX.dtype == X.dtype and dX.shape == X.shape
    assert ((dX.double() - rx).abs() <= limit).all(), float(((dX.double() - rx).abs() / limit).max())


SHAPES = [((1, 4), 1), ((2, 1, 8), 2), ((3, 5, 7, 12), 3), ((1, 16, 16, 320), 32), ((4, 9, 11, 64), 16), ((5, 13, 30), 5), ((2, 33, 17, 99), 3), ((2, 20, 20, 37), 37), ((3, 64, 6), 1),
          ((2, 7, 2048), 1), ((1, 3, 2500), 2), ((16, 32, 32, 32), 8), ((1, 128, 96, 64), 32), ((2, 1, 1, 256), 4), ((7, 40, 24), 6), ((1, 70001, 8), 2), ((130, 3, 16), 16)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,G", SHAPES)
def test_values_and_gradients(eng, dtype, shape, G):
    for i, act in enumerate(("none", "silu", "leakyRelu")):
        X, dY, gamma, beta = make(shape, dtype, i, ("same", "f32", "none")[i])
        mean, rstd = check_forward(eng, X, G, gamma, beta, act)
        check_delta(eng, X, dY, G, gamma, beta, act, mean, rstd)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", TYPES)
def test_activations(eng, dtype, act):
    for shape, G in (((2, 24, 24, 64), 8), ((2, 24, 25, 51), 17)):
        X, dY, gamma, beta = make(shape, dtype, 5, spread=4.0)
        mean, rstd = check_forward(eng, X, G, gamma, beta, act)
        check_delta(eng, X, dY, G, gamma, beta, act, mean, rstd)


@pytest.mark.parametrize("dtype", TYPES)
def test_means_far_from_zero(eng, dtype):
    """A thousand deviations from 0 in fp32 (60 in 16 bits, whose elements resolve no more), the first rows 0 as those of a padded batch."""
    for shape, G in (((2, 50, 50, 32), 4), ((2, 50, 50, 33), 3)):
        X, dY, gamma, beta = make(shape, dtype, 6, offset=1000.0 if dtype == "f32" else 60.0)
        mean, rstd = check_forward(eng, X, G, gamma, beta, "silu")
        check_delta(eng, X, dY, G, gamma, beta, "silu", mean, rstd)
        X[:, 0] = 0
        check_forward(eng, X, G, gamma, beta, "none")


@pytest.mark.parametrize("dtype", TYPES)
def test_both_routes_agree(eng, lib, dtype):
    """Large enough that the tensors are streamed, and small samples that fit into shared memory; every cluster size is met."""
    plans = set()
    for shape, G in (((1, 256, 256, 128), 32), ((512, 16, 16, 64), 32), ((64, 56, 56, 16), 4), ((32, 40, 40, 64), 2), ((300, 8, 8, 32), 4), ((24, 64, 64, 32), 8)):
        X, dY, gamma, beta = make(shape, dtype, 7)
        mean, rstd = check_forward(eng, X, G, gamma, beta, "leakyRelu")
        plans.add(lib.last_plan().split(" part")[0])
        check_delta(eng, X, dY, G, gamma, beta, "leakyRelu", mean, rstd)
        plans.add(lib.last_plan().split(" part")[0])
    assert any("streamed" in p for p in plans) and any("resident" in p for p in plans), plans


def test_constant_groups_and_eps(eng):
    X = torch.full((2, 6, 6, 16), 3.0, device="cuda")
    Y, mean, rstd = eng.groupNorm(X, 4, eps=1e-3, save=True)
    assert (Y == 0).all() and (mean == 3).all() and torch.allclose(rstd, torch.full_like(rstd, 1e-3 ** -0.5), rtol=1e-6)


def test_nan_and_inf_stay_in_their_group(eng):
    X, _, gamma, beta = make((3, 8, 8, 32), "f32", 8)
    clean = eng.groupNorm(X, 8, gamma, beta, act="silu")
    X[1, 2, 3, 5] = float("nan")
    X[2, 0, 0, 31] = float("inf")
    Y = eng.groupNorm(X, 8, gamma, beta, act="silu")
    bad = torch.zeros_like(X, dtype=torch.bool)
    bad[1, ..., 4:8] = True
    bad[2, ..., 28:32] = True
    assert torch.equal(Y[~bad], clean[~bad]) and Y[1, ..., 4:8].isnan().all() and not Y[2, ..., 28:32].isfinite().any()


def test_differences(eng):
    """The gradients against differences of the forward pass: sum(Y w) at X +- h d, in fp32 values of h that leave 64-bit differences exact to 1e-2."""
    X, w, gamma, beta = make((2, 5, 5, 12), "f32", 9)
    _, mean, rstd = eng.groupNorm(X, 3, gamma, beta, act="gelu", save=True)
    dX, dG, dB = eng.groupNorm_delta(w, X, mean, rstd, gamma, beta, act="gelu")
    h = 1e-2
    for t, grad in ((X, dX), (gamma, dG), (beta, dB)):
        d = torch.randn(t.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
        vals = []
        for sign in (1, -1):
            args = [a + sign * h * d if a is t else a for a in (X, gamma, beta)]
            vals.append(float((eng.groupNorm(args[0], 3, args[1], args[2], act="gelu").double() * w.double()).sum()))
        # third derivatives of a smooth function of unit scale over 300 elements, and 2^-23 of 300 terms over h
        assert abs((vals[0] - vals[1]) / (2 * h) - float((grad.double() * d.double()).sum())) <= 0.05 * float((grad.double().abs() * d.double().abs()).sum()) ** 0.5 + 0.02


@pytest.mark.parametrize("dtype", ("f32", "bf16"))
def test_views_and_alignment(eng, dtype):
    """Tensors that are not dense, negated views, and dense ones that start on no word's boundary."""
    base, dY, gamma, beta = make((2, 6, 10, 16), dtype, 10)
    X = base.transpose(1, 2)
    assert torch.equal(eng.groupNorm(X, 4, gamma, beta), eng.groupNorm(X.contiguous(), 4, gamma, beta))
    flat = torch.empty(base.numel() + 1, dtype=base.dtype, device="cuda")
    off = flat[1:].view(base.shape)
    off.copy_(base)
    mean, rstd = check_forward(eng, off, 4, gamma, beta, "silu")
    check_delta(eng, off, dY, 4, gamma, beta, "silu", mean, rstd)
    if dtype == "f32":
        neg = torch.complex(torch.zeros_like(base), base).conj().imag
        assert neg.is_neg() and torch.equal(eng.groupNorm(neg, 4, gamma, beta), eng.groupNorm(-base, 4, gamma, beta))


def test_other_streams_and_no_positions(eng, pkg):
    X, dY, gamma, beta = make((4, 32, 32, 64), "bf16", 11)
    want = eng.groupNorm(X, 8, gamma, beta, act="silu", save=True)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    own = pkg.submodule("engine").Engine(pkg.submodule("engine").CudaFloat32EngineBase(stream=s))
    got = own.groupNorm(X, 8, gamma, beta, act="silu", save=True)
    with torch.cuda.stream(torch.cuda.Stream()):
        more = eng.groupNorm_delta(dY, X, want[1], want[2], gamma, beta, act="silu")
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    assert all(torch.equal(a, b) for a, b in zip(more, eng.groupNorm_delta(dY, X, want[1], want[2], gamma, beta, act="silu")))
    Y, mean, rstd = eng.groupNorm(X[:0], 8, gamma, beta, save=True)
    assert Y.shape == (0, 32, 32, 64) and mean.shape == rstd.shape == (0, 8)
    dX, dG, dB = eng.groupNorm_delta(dY[:0], X[:0], mean, rstd, gamma, beta)
    assert dX.shape == Y.shape and (dG == 0).all() and (dB == 0).all()


@pytest.mark.parametrize("shape,G", [((8, 16, 16, 64), 8), ((1, 200, 200, 64), 8)])
def test_capture_and_replay(eng, lib, shape, G):
    X, dY, gamma, beta = make(shape, "bf16", 12)
    run = lambda: (lambda f: f + eng.groupNorm_delta(dY, X, f[1], f[2], gamma, beta, act="silu"))(eng.groupNorm(X, G, gamma, beta, act="silu", save=True))   # noqa: E731
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        run()
        with torch.cuda.graph(graph, stream=s):
            out = run()
    for seed in (13, 14):
        nX, ndY, ng, nb = make(shape, "bf16", seed)
        for a, b in ((X, nX), (dY, ndY), (gamma, ng), (beta, nb)):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, run()))
    assert lib.device_status() == 0


def test_workspace_and_refusals(eng, lib):
    s = lib.AlphaNormShape(4, 64 * 64, 640, 32, 1, 1, 3, 0.0, 1e-5)
    assert lib.groupNorm_workspace_bytes(s, "deltaX") >= 4 * 640 * 8 and lib.groupNorm_workspace_bytes(s, "forward") >= 0
    X, dY, gamma, beta = make((2, 4, 4, 8), "f32")
    for bad in (lambda: eng.groupNorm(X.double(), 2), lambda: eng.groupNorm(X, 3), lambda: eng.groupNorm(X, 0), lambda: eng.groupNorm(X, 2, gamma), lambda: eng.groupNorm(X, 2, gamma[:4], beta[:4]),
                lambda: eng.groupNorm(X, 2, gamma, beta.half()), lambda: eng.groupNorm(X, 2, act="relu6"), lambda: eng.groupNorm(X[:, :0], 2), lambda: eng.groupNorm(X[0, 0, 0], 2),
                lambda: eng.groupNorm(X, 2, gamma.cpu(), beta.cpu()), lambda: eng.groupNorm_delta(dY[:1], X, X.new_ones(2, 2), X.new_ones(2, 2)),
                lambda: eng.groupNorm_delta(dY, X, X.new_ones(2, 2), X.new_ones(2, 4)), lambda: eng.groupNorm_delta(dY, X, X.new_ones(2, 2).double(), X.new_ones(2, 2)),
                lambda: eng.groupNorm_delta(dY, X, X.new_ones(4), X.new_ones(4))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(lib.AlphaConvError):
        eng.groupNorm(X, 2, eps=-1.0)
    with pytest.raises(lib.AlphaConvError):
        eng.groupNorm(X, 2, act="leakyRelu", k=float("nan"))
