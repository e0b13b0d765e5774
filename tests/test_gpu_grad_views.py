"""grad_norm and clip_grad_norm over tensors that are not dense: the views that fullConnect_delta returns, columns, transposed, strided and negated ones.

Bounds as for dense tensors: the norm 5 2^-24 of itself, an element 7 2^-24 and its type's rounding."""
import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(scope="module")
def eng(pkg):
    return pkg.submodule("engine").Engine()


def norm64(grads):
    return math.sqrt(sum(float((g.double() ** 2).sum()) for g in grads))


def check(out, before, norm, max_norm):
    ref = norm64(before)
    assert abs(float(norm) - ref) <= 5 * 2.0 ** -24 * ref
    c = min(1.0, max_norm / (ref + 1e-6))
    for o, g in zip(out, before):
        want, t = g.double() * c, torch.finfo(o.dtype)
        assert ((o.double() - want).abs() <= (7 * 2.0 ** -24 + t.eps / 2) * want.abs() + t.smallest_normal * t.eps).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("glu", (False, True), ids=("fc", "glu"))
@pytest.mark.parametrize("rows,IC,OC", [(1, 700, 129), (77, 1001, 50), (300, 333, 257), (64, 72, 40)])
def test_gradients_of_a_layer_are_clipped_as_they_come(eng, dtype, glu, rows, IC, OC):
    """Forward, gradients, clipping in place, without a copy of the caller's in between."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    t, H = TYPES[dtype], 2 if glu else 1
    rand = lambda *s: torch.randn(s, device="cuda", generator=gen).to(t)
    X, W, B, dY = rand(rows, IC), (rand(H * OC, IC) * IC ** -0.5).to(t), rand(H * OC), rand(rows, OC)
    _, Z = (eng.fullConnect_glu if glu else eng.fullConnect)(X, W, B, act="silu", save=True)
    grads = (eng.fullConnect_glu_delta if glu else eng.fullConnect_delta)(dY, X, W, Z, act="silu", bias=True)
    before = [g.clone() for g in grads]
    assert abs(float(eng.grad_norm(grads)) - norm64(before)) <= 5 * 2.0 ** -24 * norm64(before)
    max_norm = 0.25 * norm64(before)
    check(grads, before, eng.clip_grad_norm(grads, max_norm), max_norm)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("out", TYPES)
def test_views_and_what_lies_between(eng, dtype, out):
    gen = torch.Generator(device="cuda").manual_seed(2)
    big = torch.randn(40, 50, device="cuda", generator=gen).to(TYPES[dtype])
    to = torch.full((40, 50), 9.0, device="cuda").to(TYPES[out])
    views = lambda t: [t[:10, :20], t[:10, 20:37], t[10:20].T, t[20:30, ::3], t[30:, :7], t[39, 8:49]]
    grads, before, kept = views(big), [g.clone() for g in views(big)], big.clone()
    max_norm = 0.5 * norm64(before)
    norm = eng.clip_grad_norm(grads, max_norm, Out=views(to))
    check(views(to), before, norm, max_norm)
    assert torch.equal(big, kept)
    mark = torch.ones(40, 50, dtype=torch.bool, device="cuda")
    for v in views(mark):
        v.zero_()
    assert (to[mark] == 9).all()
    check(grads, before, eng.clip_grad_norm(grads, max_norm), max_norm)
    assert torch.equal(big[mark], kept[mark])
    # factor 1: nothing changes; some dense, some not
    kept, dense = big.clone(), torch.ones(33, device="cuda", dtype=TYPES[dtype])
    eng.clip_grad_norm(views(big) + [dense], 1e9)
    assert torch.equal(big, kept) and (dense == 1).all()


def test_expanded_and_negated(eng):
    row = torch.arange(5.0, device="cuda")
    wide = row.expand(7, 5)
    assert abs(float(eng.grad_norm([wide])) - math.sqrt(7 * 30)) <= 1e-5
    out = torch.empty(7, 5, device="cuda")
    eng.clip_grad_norm([wide], 1.0, Out=[out])
    assert ((out - wide / math.sqrt(210)).abs() <= 1e-6).all()
    with pytest.raises(ValueError, match="share memory"):
        eng.clip_grad_norm([wide], 1.0)
    c = torch.randn(12, 16, device="cuda", dtype=torch.complex64)
    x = c.conj().imag
    assert x.is_neg()
    before = x.clone()
    check([x], [before], eng.clip_grad_norm([x], 0.5), 0.5)
    with pytest.raises(ValueError, match="overlaps"):
        big = torch.ones(4, 10, device="cuda")
        eng.clip_grad_norm([big[:, :6], big[:, 5:]], 1.0)
    assert (big == 1).all()


def test_leaves_that_require_gradients(eng):
    w = torch.randn(6, 10, device="cuda", requires_grad=True)
    before = w.detach().clone()
    check([w.detach()[:, :7]], [before[:, :7]], eng.clip_grad_norm([w[:, :7]], 0.5), 0.5)
    p = torch.nn.Parameter(torch.randn(10, 6, device="cuda").T)
    before = p.detach().clone()
    check([p.detach()], [before], eng.clip_grad_norm([p], 0.5), 0.5)


def test_own_stream_and_capture(pkg):
    engine = pkg.submodule("engine")
    s = torch.cuda.Stream()
    eng = engine.Engine(engine.CudaFloat32EngineBase(stream=s))
    big = torch.randn(1000, 1003, device="cuda")
    kept = big.clone()
    torch.cuda.synchronize()
    views = lambda t: [t[:, :700], t[:, 701:]]
    norm = eng.clip_grad_norm(views(big), 3.0)
    torch.cuda.synchronize()
    check(views(big), views(kept), norm, 3.0)
    assert torch.equal(big[:, 700], kept[:, 700])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        norm = eng.clip_grad_norm(views(big), 3.0)
    big.copy_(kept)
    torch.cuda.synchronize()
    g.replay()
    torch.cuda.synchronize()
    check(views(big), views(kept), norm, 3.0)
