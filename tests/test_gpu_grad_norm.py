"""grad_norm and clip_grad_norm against 64-bit sums.

Bounds.  The squares of a word are added in fp32 (at most 8 roundings of 2^-24 of a positive sum), everything else in fp64, and the
root halves a relative error: 4 2^-24 + the float norm's own 2^-24.  A scaled element errs by the factor's rounding and its own product's
(2 2^-24) and the output's eps / 2."""
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


def check_norm(norm, ref):
    assert norm.dtype == torch.float32 and norm.dim() == 0
    assert abs(float(norm) - ref) <= 5 * 2.0 ** -24 * ref + 1e-45


def check_scaled(out, grad, ref_norm, max_norm):
    c = min(1.0, max_norm / (ref_norm + 1e-6))
    want = grad.double() * c
    half = torch.finfo(out.dtype).eps / 2
    limit = (7 * 2.0 ** -24 + half) * want.abs() + torch.finfo(out.dtype).smallest_normal * torch.finfo(out.dtype).eps
    assert ((out.double() - want).abs() <= limit).all()


SETS = {"one": [1], "empty": [0, 5, 0], "odd": [3, 7, 8191, 8192, 8193, 1, 0, 100003], "many": [17 * i % 4001 for i in range(300)], "large": [5000000, 1000, 3000001]}


@pytest.mark.parametrize("sizes", SETS)
@pytest.mark.parametrize("dtype", TYPES)
def test_norm_and_clip(eng, dtype, sizes):
    gen = torch.Generator(device="cuda").manual_seed(3)
    grads = [torch.randn(n, device="cuda", generator=gen).mul_(0.1).to(TYPES[dtype]) for n in SETS[sizes]]
    ref = norm64(grads)
    check_norm(eng.grad_norm(grads), ref)
    for max_norm in (ref * 0.3, ref * 2 + 1):
        mine = [g.clone() for g in grads]
        check_norm(eng.clip_grad_norm(mine, max_norm), ref)
        for m, g in zip(mine, grads):
            check_scaled(m, g, ref, max_norm)
            if max_norm > ref:
                assert torch.equal(m, g)
        for other in TYPES.values():
            out = [torch.full_like(g, 7, dtype=other) for g in grads]
            check_norm(eng.clip_grad_norm(grads, max_norm, Out=out), ref)
            for o, g in zip(out, grads):
                check_scaled(o, g, ref, max_norm)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("out", TYPES)
def test_unaligned_views_leave_their_neighbours(eng, dtype, out):
    gen = torch.Generator(device="cuda").manual_seed(4)
    for at, out_at, n in ((1, 1, 20000), (3, 2, 9001), (7, 0, 5), (5, 5, 1), (0, 3, 8192), (8, 4, 16385)):
        flat = torch.randn(n + 40, device="cuda", generator=gen).to(TYPES[dtype])
        to = torch.full((n + 40,), 9.0, device="cuda").to(TYPES[out])
        g, o = flat[at:at + n], to[out_at:out_at + n]
        ref = norm64([g])
        check_norm(eng.clip_grad_norm([g], 0.5 * ref, Out=[o]), ref)
        check_scaled(o, g, ref, 0.5 * ref)
        assert (to[:out_at] == 9).all() and (to[out_at + n:] == 9).all()
        before = flat.clone()
        eng.clip_grad_norm([g], 0.5 * ref)
        check_scaled(g, before[at:at + n], ref, 0.5 * ref)
        assert torch.equal(flat[:at], before[:at]) and torch.equal(flat[at + n:], before[at + n:])


@pytest.mark.parametrize("scale", (1e-30, 1e-22, 1e-17, 1e15, 1e25, 1e36))
def test_range_of_squares(eng, scale):
    gen = torch.Generator(device="cuda").manual_seed(5)
    g = torch.randn(30000, device="cuda", generator=gen).mul_(scale)
    g[::3] = 0
    ref = norm64([g])
    check_norm(eng.grad_norm([g]), ref)
    if ref > 1:
        mine = g.clone()
        eng.clip_grad_norm([mine], 1e-3)
        check_scaled(mine, g, ref, 1e-3)


def test_not_finite(eng):
    for bad in (float("nan"), float("inf"), -float("inf")):
        a, b = torch.ones(1000, device="cuda"), torch.ones(777, device="cuda")
        b[300] = bad
        norm = float(eng.grad_norm([a, b]))
        assert math.isnan(norm) if math.isnan(bad) else norm == math.inf
        eng.clip_grad_norm([a, b], 1.0)
        # c is 0 for an infinite norm and NaN for a NaN
        assert bool(torch.isnan(a).all()) if math.isnan(bad) else bool((a == 0).all())
        assert bool(torch.isnan(b[300]))


def test_same_bits(eng):
    gen = torch.Generator(device="cuda").manual_seed(6)
    grads = [torch.randn(n, device="cuda", generator=gen) for n in (100000, 33, 2000001)]
    first = eng.grad_norm(grads)
    for _ in range(20):
        assert torch.equal(eng.grad_norm(grads), first)


def test_capture_and_replay(eng, pkg):
    lib = pkg.submodule("lib")
    grads = [torch.randn(n, device="cuda") for n in (5000, 123)]
    out = [torch.empty_like(g) for g in grads]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    lib.release_workspace()                                  # (streams come from a pool: this one may have served another test)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        with pytest.raises(lib.AlphaConvError) as e:
            eng.clip_grad_norm(grads, 1.0, Out=out)          # (no scratch yet)
        assert e.value.code == -6
    with torch.cuda.stream(s):
        eng.clip_grad_norm(grads, 1.0, Out=out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        norm = eng.clip_grad_norm(grads, 1.0, Out=out)
    for a in grads:
        a.mul_(3.0)
    torch.cuda.synchronize()
    g.replay()
    torch.cuda.synchronize()
    ref = norm64(grads)
    check_norm(norm, ref)
    for o, a in zip(out, grads):
        check_scaled(o, a, ref, 1.0)


def test_nothing_to_do(eng):
    assert float(eng.grad_norm([])) == 0 and float(eng.clip_grad_norm([], 1.0)) == 0
    empty = torch.empty(0, device="cuda")
    assert float(eng.grad_norm([empty])) == 0 and float(eng.clip_grad_norm([empty, empty], 1.0)) == 0
    zeros = torch.zeros(100000, device="cuda")
    assert float(eng.clip_grad_norm([zeros], 1.0)) == 0 and not zeros.any()
    ones = torch.ones(10, device="cuda")
    eng.clip_grad_norm([ones], 0.0)
    assert not ones.any()
    ones = torch.ones(10, device="cuda")
    eng.clip_grad_norm([ones], float("inf"))
    assert (ones == 1).all()


def test_more_than_2_31_elements(eng):
    big = torch.full((2 ** 31 + 12345,), 2.0 ** -10, device="cuda", dtype=torch.bfloat16)
    big[-1] = 3.0
    ref = math.sqrt((big.numel() - 1) * 2.0 ** -20 + 9.0)
    check_norm(eng.clip_grad_norm([big], ref / 2), ref)
    half = 2.0 ** -11 * (ref / (ref + 1e-6))
    for at in (0, 2 ** 31 - 1, 2 ** 31, big.numel() - 2):
        assert abs(float(big[at]) - half) <= 2.0 ** -8 * half
    assert abs(float(big[-1]) - 1.5) <= 2.0 ** -7


@pytest.mark.parametrize("max_norm", (1.0, 0.37, 1e-3, 1e-25, 123.456))
@pytest.mark.parametrize("n", (3, 10001))
def test_a_product_is_rounded_once(eng, n, max_norm):
    """Gradients whose squares sum without rounding: the factor is that of fp64, and an fp32 output errs by its own rounding only (2^-24, and 2^-47 of the
    factor's two floats; of the smallest by the denormals' spacing)."""
    gen = torch.Generator(device="cuda").manual_seed(n)
    g = torch.randint(-200, 201, (n,), device="cuda", generator=gen).float() / 64
    for t in (torch.float32, torch.bfloat16):
        grad, out = g.to(t), torch.empty_like(g)
        c = min(1.0, max_norm / (math.sqrt(float((grad.double() ** 2).sum())) + 1e-6))
        eng.clip_grad_norm([grad], max_norm, Out=[out])
        want = grad.double() * c
        assert ((out.double() - want).abs() <= 2.0 ** -24 * (1 + 2.0 ** -20) * want.abs() + 2.0 ** -149).all()
