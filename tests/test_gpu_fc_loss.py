"""fullConnect_softmax_crossEntropy and its gradients against 64-bit results.

Bounds, with e = 2^-24 and u = eps / 2 of the type.  A logit is a sum of IC products in fp32; the tensor cores truncate as they add 16 at a time: (IC / 16 + 8) 2 e of the sum
of its terms' magnitudes (fp32 tensors, three bf16 planes: twice as many steps and 8 e more), and the bias's addition e of the result.  lse errs by the largest such error, and by
64 e (1 + |lse|) for exponentials, their sum and the logarithm.  A probability errs by itself times its logit's and lse's errors and 2^-20.  dz = dL (p - [label]) is rounded
to the tensors' type (16 bits: u), and deltaX, deltaW, deltaB err by the sum of their terms' errors, by (terms / 16 + 24) 2 e of the sum of their magnitudes, and their own rounding."""
import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
E = 2.0 ** -24


@pytest.fixture(scope="module")
def eng(pkg):
    return pkg.submodule("engine").Engine()


@pytest.fixture(scope="module")
def lib(pkg):
    return pkg.submodule("lib")


def make(rows, IC, OC, dtype, bias=True, ignored=0.2, seed=0, scale=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = TYPES[dtype]
    W = (torch.randn(OC, IC, device="cuda", generator=g) * scale / math.sqrt(IC)).to(t)
    label = torch.randint(0, OC, (rows,), device="cuda", generator=g)
    X = (torch.randn(rows, IC, device="cuda", generator=g) + torch.rand(rows, 1, device="cuda", generator=g) * 2 * W[label].float()).to(t)
    label[torch.rand(rows, device="cuda", generator=g) < ignored] = -1
    B = (torch.randn(OC, device="cuda", generator=g) * 0.5).to(t) if bias else None
    return X, W, label, B


def logits(X, W, B):
    x, w = X.double().reshape(-1, X.shape[-1]), W.double()
    z = x @ w.T + (0 if B is None else B.double())
    steps = (X.shape[-1] / 16 + 8) * 2 if X.dtype != torch.float32 else (X.shape[-1] / 8 + 12) * 2
    return z, steps * E * (x.abs() @ w.abs().T) + 2 * E * z.abs().nan_to_num(posinf=0.0)


def check(eng, X, W, label, B, dL=None, grads=True):
    loss, lse = eng.fullConnect_softmax_crossEntropy(X, W, label, B, save=True)
    z, zerr = logits(X, W, B)
    counts = ((label >= 0) & (label < W.shape[0])).reshape(-1)
    at = torch.where(counts, label.reshape(-1), 0).long()[:, None]
    want = torch.logsumexp(z, 1)
    worst = zerr.max(1).values
    limit = worst + 64 * E * (1 + want.abs())
    assert loss.dtype == lse.dtype == torch.float32 and loss.shape == lse.shape == label.shape
    assert ((lse.reshape(-1).double() - want).abs() <= limit).all()
    wl = torch.where(counts, want - z.gather(1, at)[:, 0], torch.zeros_like(want))
    ll = torch.where(counts, limit + zerr.gather(1, at)[:, 0] + 2 * E * z.gather(1, at)[:, 0].abs(), torch.zeros_like(want))
    assert ((loss.reshape(-1).double() - wl).abs() <= ll).all()
    assert torch.equal(loss, eng.fullConnect_softmax_crossEntropy(X, W, label, B))
    if not grads:
        return loss, lse
    rows = X.reshape(-1, X.shape[-1]).shape[0]
    if dL is None:
        dL = torch.rand(label.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)) + 0.5
    out = eng.fullConnect_softmax_crossEntropy_delta(dL, X, W, label, lse, B)
    again = eng.fullConnect_softmax_crossEntropy_delta(dL, X, W, label, lse, B)
    assert all(a is b or torch.equal(a, b) for a, b in zip(out, again))
    d = (dL.double() if isinstance(dL, torch.Tensor) else torch.tensor(dL, dtype=torch.float64, device="cuda")).reshape(-1).expand(rows) * counts
    p = torch.exp(z - want[:, None])
    one = torch.zeros_like(p)
    one[counts, at[counts, 0]] = 1.0
    dz = torch.where(counts[:, None], d[:, None] * (p - one), torch.zeros_like(p))
    u = 0.0 if X.dtype == torch.float32 else torch.finfo(X.dtype).eps / 2
    perr = p * (zerr + limit[:, None] + 2.0 ** -20) + 4 * E * (p + one)
    dzerr = torch.where(counts[:, None], d.abs()[:, None] * perr, torch.zeros_like(p)) + (u + 2 * E) * dz.abs()
    if X.dtype == torch.float16:
        dzerr = dzerr + d.abs().max() * 2.0 ** -38 * counts[:, None]         # half a step of a denormal, 2^-24 of a scale that has the largest |dL| at 2^14 or above
    x, w = X.double().reshape(rows, -1), W.double()
    half = torch.finfo(X.dtype).eps / 2
    tiny = torch.finfo(X.dtype).smallest_normal * (torch.finfo(X.dtype).eps if X.dtype != torch.float32 else 1)
    for name, got, ref, err, mags, terms in (("X", out[0], dz @ w, dzerr @ w.abs(), dz.abs() @ w.abs(), W.shape[0]), ("W", out[1], dz.T @ x, dzerr.T @ x.abs(), dz.abs().T @ x.abs(), rows),
                                             ("B", out[2], dz.sum(0), dzerr.sum(0), dz.abs().sum(0), rows)):
        if name == "B" and B is None:
            assert got is None
            continue
        bound = err + (terms / 16 + 24) * 4 * E * mags + half * ref.abs() + tiny
        off = (got.double().reshape(ref.shape) - ref).abs()
        assert got.dtype == X.dtype and (off <= bound).all(), (name, float((off / bound).max()))
    return loss, lse, out


SHAPES = [(1, 8, 1), (1, 64, 10), (3, 40, 33), (5, 17, 259), (16, 96, 1000), (65, 72, 100), (129, 256, 1001), (300, 1001, 517), (1000, 128, 4099), (257, 512, 20000), (2, 2048, 30011), (4, 4096, 512)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_values_and_gradients(eng, lib, dtype, shape):
    for bias, ignored in ((True, 0.3), (False, 0.0)):
        check(eng, *make(*shape, dtype, bias, ignored))
    assert lib.device_status() == 0


@pytest.mark.parametrize("shape", ((1, 40, 3001), (2, 72, 9000), (13, 64, 40001), (100, 24, 6000), (256, 8, 300000)))
def test_few_rows_of_many_classes_in_f32(eng, lib, shape):
    """Several CTAs to a row, of one piece of the classes or of two (the last shape), and shares of a row that hold masked classes only."""
    X, W, label, B = make(*shape, "f32")
    check(eng, X, W, label, B)
    B[5:] = -float("inf")
    label.clamp_(-1, 4)
    check(eng, X, W, label, B)
    assert lib.device_status() == 0


@pytest.mark.parametrize("tile", (0, 1, 11))
@pytest.mark.parametrize("shape", ((256, 512, 1000), (300, 700, 501), (513, 512, 1000), (1024, 130, 263), (2048, 512, 1000)))
def test_both_gradients_by_one_launch_in_f32(eng, lib, shape, tile):
    """Shapes whose deltaX and deltaW one launch makes, whole and in parts of either, and columns so small and so large that the planes do not hold the products."""
    old = lib.set_option("FC_TILE", tile)
    try:
        X, W, label, B = make(*shape, "f32")
        check(eng, X, W, label, B)
        X[:, :8] *= 1e-36
        X[:, 8:16] *= 1e-30
        W[:, 8:16] *= 1e30
        check(eng, X, W, label, B)
    finally:
        lib.set_option("FC_TILE", old)
    assert lib.device_status() == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tile", (1, 11, 1064, 1128, 2064, 4256))
def test_every_tile(eng, lib, dtype, tile):
    """Kernels chosen by hand: pairs of 256 and 128 columns, tiles of 64 and 128, and requests for shared or wider tiles than these epilogues take."""
    old = lib.set_option("FC_TILE", tile)
    try:
        check(eng, *make(200, 2100 if dtype != "f32" else 300, 700, dtype))
    finally:
        lib.set_option("FC_TILE", old)


@pytest.mark.parametrize("dtype", TYPES)
def test_several_pieces(eng, dtype):
    """More logits than one piece of scratch holds: 256 MB are 134 million of 16 bits, 67 million of fp32."""
    rows, OC = (9000, 16500) if dtype != "f32" else (4100, 17000)
    X, W, label, B = make(rows, 32, OC, dtype, True, 0.1)
    loss, lse = eng.fullConnect_softmax_crossEntropy(X, W, label, B, save=True)
    dX, dW, dB = eng.fullConnect_softmax_crossEntropy_delta(1.0, X, W, label, lse, B)
    half, u = torch.finfo(X.dtype).eps / 2, 0.0 if dtype == "f32" else torch.finfo(X.dtype).eps / 2
    rdW, rdB, ldW, ldB = 0.0, 0.0, 0.0, 0.0
    for part in torch.arange(rows, device="cuda").split(1500):
        x, l = X[part], label[part]
        z, zerr = logits(x, W, B)
        want = torch.logsumexp(z, 1)
        limit = zerr.max(1).values + 64 * E * (1 + want.abs())
        assert ((lse[part].double() - want).abs() <= limit).all()
        counts = l >= 0
        p = torch.exp(z - want[:, None])
        dz = p.clone()
        dz[counts, l[counts]] -= 1
        dz[~counts] = 0
        err = (p * (zerr + limit[:, None] + 2.0 ** -20) + 8 * E) * counts[:, None] + (u + 2.0 ** -24 * (dtype == "f16")) * dz.abs()
        w = W.double()
        off = (dX[part].double() - dz @ w).abs()
        assert (off <= err @ w.abs() + (OC / 16 + 24) * 4 * E * (dz.abs() @ w.abs()) + half * (dz @ w).abs() + 1e-7).all()
        xd = x.double()
        rdW, rdB = rdW + dz.T @ xd, rdB + dz.sum(0)
        ldW, ldB = ldW + (err + 1200 * E * dz.abs()).T @ xd.abs(), ldB + (err + 1200 * E * dz.abs()).sum(0)
    assert ((dW.double() - rdW).abs() <= ldW + half * rdW.abs() + 1e-7).all()
    assert ((dB.double() - rdB).abs() <= ldB + half * rdB.abs() + 1e-7).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_forms_of_the_losses_gradient(eng, dtype):
    X, W, label, B = make(70, 64, 300, dtype)
    _, lse = eng.fullConnect_softmax_crossEntropy(X, W, label, B, save=True)
    number = eng.fullConnect_softmax_crossEntropy_delta(0.25, X, W, label, lse, B)
    value = eng.fullConnect_softmax_crossEntropy_delta(torch.tensor(0.25, device="cuda"), X, W, label, lse, B)
    assert all(torch.equal(a, b) for a, b in zip(number, value))
    check(eng, X, W, label, B, 0.25)
    check(eng, X, W, label, B, torch.full((70,), 0.25, device="cuda"))
    # gradients of very different sizes, of both signs, zeros among them; of a mean over many rows
    g = torch.Generator(device="cuda").manual_seed(3)
    dL = torch.randn(70, device="cuda", generator=g) * torch.tensor([1.0, 0.0, 1e-3, 3.0], device="cuda").repeat(18)[:70]
    check(eng, X, W, label, B, dL)
    check(eng, X, W, label, B, 0.0)
    if dtype != "f16":
        check(eng, X, W, label, B, 1e-9)


def test_small_probabilities_in_fp16(eng):
    """dL of 1 / 30000 and probabilities of 1e-4: products near 3e-9, no fp16 numbers, whose sums over the rows of deltaB and deltaW are."""
    X, W, label, B = make(4000, 64, 9000, "f16", True, 0.0, scale=0.3)
    check(eng, X, W, label, B, 1 / 3e4)


@pytest.mark.parametrize("dtype", TYPES)
def test_gradients_of_losses_that_do_not_count(eng, dtype):
    """Inf, NaN and huge gradients of losses that do not count change nothing: not the scale of fp16 either."""
    X, W, label, B = make(100, 64, 3000, dtype, True, 0.3, scale=0.3)
    _, lse = eng.fullConnect_softmax_crossEntropy(X, W, label, B, save=True)
    dL = torch.full((100,), 1e-4, device="cuda")
    want = eng.fullConnect_softmax_crossEntropy_delta(dL, X, W, label, lse, B)
    out = (label < 0).nonzero()[:, 0]
    assert out.numel() > 4
    dL[out] = 1e30
    dL[out[0]], dL[out[1]] = float("inf"), float("nan")
    assert all(torch.equal(a, b) for a, b in zip(want, eng.fullConnect_softmax_crossEntropy_delta(dL, X, W, label, lse, B)))


@pytest.mark.parametrize("dtype", TYPES)
def test_masked_classes(eng, dtype):
    """Classes with a bias of -Inf, and of the type's lowest value, have no probability; a row that counts none of its classes has an lse of -Inf."""
    X, W, label, B = make(40, 64, 200, dtype, True, 0.0)
    B[100:] = -float("inf")
    B[90:100] = torch.finfo(B.dtype).min
    label %= 90
    loss, lse = eng.fullConnect_softmax_crossEntropy(X, W, label, B, save=True)
    few = eng.fullConnect_softmax_crossEntropy(X, W[:90].contiguous(), label, B[:90].contiguous(), save=True)
    assert torch.allclose(loss, few[0], rtol=1e-5, atol=1e-5) and torch.allclose(lse, few[1], rtol=1e-5)
    dX, dW, dB = eng.fullConnect_softmax_crossEntropy_delta(1.0, X, W, label, lse, B)
    assert dX.isfinite().all() and (dW[90:] == 0).all() and (dB[90:] == 0).all() and not (dW[:90] == 0).all()
    label[3] = 150                                 # a class without probability: an infinite loss, a finite gradient
    loss = eng.fullConnect_softmax_crossEntropy(X, W, label, B)
    assert loss[3] == float("inf") and loss[torch.arange(40, device="cuda") != 3].isfinite().all()
    B[:] = -float("inf")
    _, lse = eng.fullConnect_softmax_crossEntropy(X, W, label, B, save=True)
    assert (lse == -float("inf")).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_that_do_not_count(eng, dtype):
    """Labels of -1, of OC and beyond, of -100 and of the integers' ends; NaN in such a row stays there."""
    X, W, label, B = make(50, 64, 100, dtype, True, 0.0)
    clean = label.clone()
    label[:8] = torch.tensor([-1, 100, -100, 2 ** 31 - 1, -2 ** 31, 2 ** 40, -2 ** 63, 101], device="cuda")
    loss, lse, out = check(eng, X, W, label, B)
    assert (loss[:8] == 0).all() and (out[0][:8] == 0).all() and lse.isfinite().all()
    ints = label.clamp(-2 ** 31, 2 ** 31 - 1).int()
    assert torch.equal(loss, eng.fullConnect_softmax_crossEntropy(X, W, ints, B))
    X[2] = float("nan")
    again, kept = eng.fullConnect_softmax_crossEntropy(X, W, ints, B, save=True)
    assert (again[2] == 0) and kept[2].isnan()
    # (an fp32 product forms the sums of a tile that holds a NaN in another order: either result errs by at most the bound above, so that they differ by twice that at most)
    _, zerr = logits(X[8:], W, B)
    assert ((again[8:].double() - loss[8:].double()).abs() <= 2 * (2 * zerr.max(1).values + 64 * E * (1 + lse[8:].double().abs()) + 2 * E * (loss[8:] + lse[8:].abs()))).all()
    assert dtype == "f32" or torch.equal(again[8:], loss[8:])
    dX, dW, dB = eng.fullConnect_softmax_crossEntropy_delta(1.0, X, W, ints, kept, B)
    assert (dX[:8] == 0).all() and dB.isfinite().all()       # (dW sums 0 * NaN of that row's X)
    none = torch.full_like(clean, -1)
    loss, lse, out = check(eng, make(50, 64, 100, dtype)[0], W, none, B)
    assert (loss == 0).all() and all((t == 0).all() for t in out)


def test_leading_dimensions_views_and_types_of_labels(eng):
    X, W, label, B = make(60, 50, 90, "bf16")
    want = eng.fullConnect_softmax_crossEntropy(X, W, label, B, save=True)
    got = eng.fullConnect_softmax_crossEntropy(X.view(3, 4, 5, 50), W, label.view(3, 4, 5).int(), B, save=True)
    assert all(torch.equal(a.view(3, 4, 5), b) for a, b in zip(want, got))
    out = eng.fullConnect_softmax_crossEntropy_delta(torch.ones(3, 4, 5, device="cuda"), X.view(3, 4, 5, 50), W, label.view(3, 4, 5), got[1], B)
    assert out[0].shape == (3, 4, 5, 50) and out[1].shape == W.shape and out[2].shape == B.shape
    wide = torch.cat([X, X], 1)[:, :50]
    every = torch.stack([label, label], 1)[:, 0]
    assert not wide.is_contiguous() and not every.is_contiguous()
    assert torch.equal(want[0], eng.fullConnect_softmax_crossEntropy(wide, W.t().contiguous().t(), every, B))
    one = eng.fullConnect_softmax_crossEntropy(X[0], W, label[0], B, save=True)
    assert one[0].shape == () and torch.allclose(one[1], want[1][0], rtol=1e-6)
    loss, lse = eng.fullConnect_softmax_crossEntropy(X[:0], W, label[:0], B, save=True)
    assert loss.shape == lse.shape == (0,)
    dX, dW, dB = eng.fullConnect_softmax_crossEntropy_delta(1.0, X[:0], W, label[:0], lse, B)
    assert dX.shape == (0, 50) and (dW == 0).all() and (dB == 0).all()


def test_differences(eng):
    """The gradients against differences of the summed loss along random directions, in fp32."""
    X, W, label, B = make(20, 24, 30, "f32")
    _, lse = eng.fullConnect_softmax_crossEntropy(X, W, label, B, save=True)
    grads = eng.fullConnect_softmax_crossEntropy_delta(1.0, X, W, label, lse, B)
    h = 1e-2
    for k, t in enumerate((X, W, B)):
        d = torch.randn(t.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))
        vals = [float(eng.fullConnect_softmax_crossEntropy(*[a + s * h * d if a is t else a for a in (X, W)], label, B + s * h * d if t is B else B).double().sum()) for s in (1, -1)]
        slope = float((grads[k].double() * d.double()).sum())
        # h^2 / 6 of a third derivative: that of a row's loss along d is at most the cube of its logits' range, some 10^3 for X and W here; 2^-22 of the losses over h
        assert abs((vals[0] - vals[1]) / (2 * h) - slope) <= 20 * h * h / 6 * 300 + 0.02


def test_other_streams_and_capture(eng, lib, pkg):
    X, W, label, B = make(200, 128, 1000, "bf16", True, 0.2)
    want = eng.fullConnect_softmax_crossEntropy(X, W, label, B, save=True)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    own = pkg.submodule("engine").Engine(pkg.submodule("engine").CudaFloat32EngineBase(stream=s))
    got = own.fullConnect_softmax_crossEntropy(X, W, label, B, save=True)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    dL = torch.full((), 1 / 200, device="cuda")
    run = lambda e: (lambda f: f + e.fullConnect_softmax_crossEntropy_delta(dL, X, W, label, f[1], B))(e.fullConnect_softmax_crossEntropy(X, W, label, B, save=True))   # noqa: E731
    graph, c = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    c.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(c):
        run(eng)
        with torch.cuda.graph(graph, stream=c):
            out = run(eng)
    for seed in (5, 6):
        for a, b in zip((X, W, label, B), make(200, 128, 1000, "bf16", True, 0.2, seed)):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, run(eng)))
    assert lib.device_status() == 0


def test_scratch_is_what_was_asked_for(eng, lib):
    """The bytes that the size function names are enough as a block of the caller's, and one byte of scratch is not."""
    for dtype, code in (("bf16", 1), ("f16", 2), ("f32", 0)):
        X, W, label, B = make(300, 64, 1000, dtype)
        shape = lib.AlphaFcShape(300, 64, 1000, code, 0, 0.0)
        want = eng.fullConnect_softmax_crossEntropy(X, W, label, B, save=True)
        s = torch.cuda.Stream()
        torch.cuda.synchronize()
        for op in ("forward", "deltaX"):
            n = lib.fullConnect_softmax_crossEntropy_workspace_bytes(shape, op)
            block = torch.empty(n, dtype=torch.uint8, device="cuda")
            torch.cuda.synchronize()
            with torch.cuda.stream(s):
                lib.set_workspace(s.cuda_stream, block.data_ptr(), n)
                try:
                    if op == "forward":
                        got = eng.fullConnect_softmax_crossEntropy(X, W, label, B, save=True)
                        s.synchronize()
                        assert all(torch.equal(a, b) for a, b in zip(got, want))
                    else:
                        eng.fullConnect_softmax_crossEntropy_delta(1.0, X, W, label, want[1], B)
                    lib.set_workspace(s.cuda_stream, block.data_ptr(), 256)
                    with pytest.raises(lib.AlphaConvError) as e:
                        if op == "forward":
                            eng.fullConnect_softmax_crossEntropy(X, W, label, B)
                        else:
                            eng.fullConnect_softmax_crossEntropy_delta(1.0, X, W, label, want[1], B)
                    assert e.value.code == -5
                finally:
                    s.synchronize()
                    lib.set_workspace(s.cuda_stream, 0, 0)


def test_refusals(eng, lib):
    X, W, label, B = make(20, 32, 40, "bf16")
    _, lse = eng.fullConnect_softmax_crossEntropy(X, W, label, B, save=True)
    for bad in (lambda: eng.fullConnect_softmax_crossEntropy(X, W, label.float(), B), lambda: eng.fullConnect_softmax_crossEntropy(X, W, label[:10], B),
                lambda: eng.fullConnect_softmax_crossEntropy(X, W[:, :16], label, B), lambda: eng.fullConnect_softmax_crossEntropy(X, W, label, B[:8]),
                lambda: eng.fullConnect_softmax_crossEntropy(X, W.float(), label, B), lambda: eng.fullConnect_softmax_crossEntropy(X, W, label.cpu(), B),
                lambda: eng.fullConnect_softmax_crossEntropy(X.double(), W.double(), label), lambda: eng.fullConnect_softmax_crossEntropy_delta(lse[:5], X, W, label, lse, B),
                lambda: eng.fullConnect_softmax_crossEntropy_delta(lse.double(), X, W, label, lse, B), lambda: eng.fullConnect_softmax_crossEntropy_delta(1.0, X, W, label, lse.half(), B),
                lambda: eng.fullConnect_softmax_crossEntropy_delta(torch.tensor(1.0), X, W, label, lse, B), lambda: eng.fullConnect_softmax_crossEntropy_delta(1.0, X, W, label, lse[:7], B)):
        with pytest.raises(ValueError):
            bad()


def test_a_training_step(eng):
    """Convolution, group norm, FullConnect loss, all gradients and the update, one after the other: the gradients against automatic differentiation in 64 bits (each
    fp32 operator errs by 1e-5 or less of its result's norm, and there are nine of them), and a step that moves the parameters as the formula says."""
    g = torch.Generator(device="cuda").manual_seed(8)
    rand = lambda *s, k=1.0: torch.randn(s, device="cuda", generator=g) * k      # noqa: E731
    X, Wc = rand(8, 12, 12, 8), rand(16, 3, 3, 8, k=0.1)
    gamma, beta = 1 + rand(16, k=0.1), rand(16, k=0.1)
    Wf, Bf = rand(10, 12 * 12 * 16, k=0.02), rand(10, k=0.1)
    label = torch.randint(0, 10, (8,), device="cuda", generator=g)
    conv = eng.conv3D(X, Wc, 1, 1, 1, 1)
    act, mean, rstd = eng.groupNorm(conv, 4, gamma, beta, act="silu", save=True)
    flat = act.reshape(8, -1)
    loss, lse = eng.fullConnect_softmax_crossEntropy(flat, Wf, label, Bf, save=True)
    dF, dWf, dBf = eng.fullConnect_softmax_crossEntropy_delta(1 / 8, flat, Wf, label, lse, Bf)
    dC, dG, dB = eng.groupNorm_delta(dF.reshape(act.shape).contiguous(), conv, mean, rstd, gamma, beta, act="silu")
    dWc = eng.dconv3D_deltaW(X, dC, 3, 3, 1, 1, 1, 1)
    params, grads = [Wc, gamma, beta, Wf, Bf], [dWc, dG, dB, dWf, dBf]

    leaves = [p.double().requires_grad_() for p in params]
    y = torch.nn.functional.conv2d(X.double().permute(0, 3, 1, 2), leaves[0].permute(0, 3, 1, 2), padding=1)
    y = torch.nn.functional.silu(torch.nn.functional.group_norm(y, 4, leaves[1], leaves[2])).permute(0, 2, 3, 1).reshape(8, -1)
    want = torch.nn.functional.cross_entropy(y @ leaves[3].T + leaves[4], label)
    refs = torch.autograd.grad(want, leaves)
    assert abs(float(loss.mean()) - float(want.detach())) <= 1e-4 * float(want.detach())
    for got, ref in zip(grads, refs):
        assert float((got.double() - ref).norm()) <= 9e-5 * float(ref.norm())
    before = [p.clone() for p in params]
    state = eng.adamW_state(params)
    norm = eng.adamW(params, grads, state, 1, 1e-2, weight_decay=0.0, max_norm=1e9)
    total = math.sqrt(sum(float((t.double() ** 2).sum()) for t in grads))
    assert abs(float(norm) - total) <= 1e-6 * total
    for p0, p1, t in zip(before, params, grads):
        # the first step is lr g / (|g| + eps): its sign, one rate long
        big = t.abs() > 1e-5
        assert torch.allclose((p0 - p1)[big], 1e-2 * torch.sign(t)[big], rtol=2e-3, atol=1e-6)


def test_two_streams_at_once_and_fewer_sms(eng, lib, pkg):
    """A whole step of these operators on each of two streams, enqueued in turn, and on 100 of the SMs: the same results as one after the other on all."""
    g = torch.Generator(device="cuda").manual_seed(9)
    X, W, label, B = make(300, 256, 2000, "bf16")
    N = (torch.randn(4, 40, 40, 64, device="cuda", generator=g)).bfloat16()
    big = torch.randn(1, 200, 200, 96, device="cuda", generator=g).bfloat16()
    p = torch.randn(100000, device="cuda", generator=g)

    def step(e):
        out = []
        for t, groups in ((N, 8), (big, 6)):
            y, mean, rstd = e.groupNorm(t, groups, act="silu", save=True)
            out += [y, mean, rstd, e.groupNorm_delta(y, t, mean, rstd, act="silu")[0]]
        loss, lse = e.fullConnect_softmax_crossEntropy(X, W, label, B, save=True)
        out += [loss, lse, *e.fullConnect_softmax_crossEntropy_delta(0.01, X, W, label, lse, B)]
        q, state = p.clone(), e.adamW_state([p], 8)
        e.adamW([q], [p], state, 1, 1e-2, max_norm=1.0)
        return out + [q, state.m[0].view(torch.uint8), state.v[0].view(torch.uint8)]

    want = step(eng)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = step(eng)
    torch.cuda.synchronize()
    for each in got:
        assert all(torch.equal(a, b) for a, b in zip(want, each))
    old = lib.set_option("SM_BUDGET", 100)
    try:
        few = step(eng)
    finally:
        lib.set_option("SM_BUDGET", old)
    # (other plans: other orders of summation; outputs of 16 bits a rounding apart at most where these meet a border)
    for a, b in zip(want, few):
        if a.dtype == torch.uint8:
            assert float((a != b).float().mean()) < 1e-3
        else:
            assert float((a.double() - b.double()).norm()) <= 2e-3 * float(a.double().norm())
    assert lib.device_status() == 0
