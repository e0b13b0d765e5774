"""adamW against the formula in 64 bits, and the codes of 8-bit moments against the same arithmetic in torch.

Bounds, with e = 2^-24: m is a sum of two products, each rounded, of rounded factors: 4 e of |b1 m| + |(1 - b1) g| (the factor c of a clipped gradient and its product 2 e
more); v likewise, 8 e of its terms.  The update lr m / (sqrt(v) + eps) errs by half of v's error, m's, and 2^-20 for root, quotient and products; p by 3 e |p| and its own rounding."""
import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
E = 2.0 ** -24
LR, B1, B2, EPS, WD = 1e-2, 0.9, 0.999, 1e-8, 0.05


@pytest.fixture(scope="module")
def eng(pkg):
    return pkg.submodule("engine").Engine()


@pytest.fixture(scope="module")
def lib(pkg):
    return pkg.submodule("lib")


def normal(gen, n, scale, t=torch.float32):
    return torch.randn(n, device="cuda", generator=gen).mul_(scale).to(t)


def mix(x):
    x = ((x ^ (x >> 16)) * 0x9E3779B9) & 0xFFFFFFFF
    x = ((x ^ (x >> 15)) * 0xB7E15163) & 0xFFFFFFFF
    return x ^ (x >> 16)


def random_bits(n, tensor, step, seed):
    one = lambda v: torch.tensor([v], dtype=torch.int64)      # noqa: E731
    key = mix(mix(one(0x243F6A88) ^ mix(one(seed)) ^ (step & 0xFFFFFFFF)) ^ tensor)
    return mix(torch.arange(n, dtype=torch.int64) ^ key).cuda()


def decode(codes, scales):
    return codes.reshape(-1).float() * scales.float().repeat_interleave(32)[: codes.numel()]


def encode(x, bits, floor):
    """(codes as floats, scales as exponent bytes) of a flat fp32 tensor."""
    n = x.numel()
    most = torch.nn.functional.pad(x.abs(), (0, -n % 32)).reshape(-1, 32).max(1).values
    raw = most.view(torch.int32)
    byte = ((raw >> 23) - 8 + ((raw & 0x7FFFFF) > 0x600000).int()).clamp(min=1)
    y = x * ((254 - byte) << 23).view(torch.float32).repeat_interleave(32)[:n]
    a = y.abs()
    small = a < 2.0 ** -6
    a = torch.where(small, a + 2.0 ** -6, a)
    a = ((a.view(torch.int32) + (bits << 4).int()) & ~0xFFFFF).view(torch.float32)
    a = torch.where(small, a - 2.0 ** -6, a)
    if floor:
        a = torch.where(y > 0, a.clamp(min=2.0 ** -9), a)
    return torch.copysign(a, y), byte


def check_step(p0, g, m0, v0, p1, step, wd=WD, c=1.0, lr=LR, clipped=0.0):
    """p1 against the formula from p0, g and the moments before (64-bit values); returns m and v in 64 bits with their bounds."""
    g = g.double().reshape(-1) * c
    m = B1 * m0 + (1 - B1) * g
    v = B2 * v0 + (1 - B2) * g * g
    me = (4 + clipped) * E * ((B1 * m0).abs() + ((1 - B1) * g).abs())
    ve = (8 + 2 * clipped) * E * v
    by = (v / (1 - B2 ** step)).sqrt() + EPS
    want = p0.double().reshape(-1) * (1 - lr * wd) - lr / (1 - B1 ** step) * m / by
    size = lr / (1 - B1 ** step) / by
    half = torch.finfo(p1.dtype).eps / 2
    limit = size * (me + m.abs() * (2.0 ** -20 + (8 + 2 * clipped) * E)) + (3 * E + half) * want.abs() + 3 * E * p0.double().reshape(-1).abs() + torch.finfo(p1.dtype).smallest_normal
    err = (p1.double().reshape(-1) - want).abs()
    assert (err <= limit).all(), float((err / limit).max())
    return m, v, me, ve, want


SETS = {"one": [1], "empty": [0, 5, 0], "odd": [3, 31, 32, 33, 4095, 4096, 4097, 100003], "many": [17 * i % 401 for i in range(300)], "large": [3000000, 1000, 1000001]}


@pytest.mark.parametrize("bits", (32, 8))
@pytest.mark.parametrize("sizes", SETS)
def test_steps(eng, sizes, bits):
    gen = torch.Generator(device="cuda").manual_seed(1)
    kinds = list(TYPES.values())
    params = [normal(gen, n, 0.1, kinds[i % 3]) for i, n in enumerate(SETS[sizes])]
    outs = [torch.empty_like(p, dtype=torch.bfloat16) if i % 2 else None for i, p in enumerate(params)]
    state = eng.adamW_state(params, bits)
    decay = [WD * (i % 2) for i in range(len(params))]
    for step in (1, 2, 50):
        grads = [normal(gen, p.numel(), 1e-2, kinds[(i // 3) % 3]) for i, p in enumerate(params)]
        if bits == 32:
            old = [(m.double(), v.double()) for m, v in zip(state.m, state.v)]
        else:
            old = [tuple(decode(c, s).double() for c, s in ((state.m[i], state.m_scale[i]), (state.v[i], state.v_scale[i]))) for i in range(len(params))]
        before = [p.clone() for p in params]
        assert eng.adamW(params, grads, state, step, LR, B1, B2, EPS, decay, Out=outs, seed=7) is None
        for i, (p0, p1, g, (m0, v0)) in enumerate(zip(before, params, grads, old)):
            m, v, me, ve, want = check_step(p0, g, m0, v0, p1, step, decay[i])
            if outs[i] is not None and p1.dtype == torch.float32:
                assert torch.equal(outs[i], p1.bfloat16())
            if bits == 32:
                assert ((state.m[i].double() - m).abs() <= me).all() and ((state.v[i].double() - v).abs() <= ve).all()
            elif p1.numel():
                m32 = m0.float() * B1 + g.float() * (1 - B1)
                v32 = v0.float() * B2 + (g.float() * g.float()) * (1 - B2)
                r = random_bits(p1.numel(), i, step, 7)
                for x, codes, scales, rr, floor in ((m32, state.m[i], state.m_scale[i], r & 0xFFFF, False), (v32, state.v[i], state.v_scale[i], r >> 16, True)):
                    a, byte = encode(x, rr, floor)
                    assert torch.equal(codes.float(), a) and torch.equal(scales.view(torch.uint8).int(), byte)


def test_codes_keep_their_mean(eng):
    """2^18 equal elements beside one that sets the scale: the mean of their codes is the element's value within five deviations of a rounding up or down at random,
    and one that is not 0 has no code of 0."""
    n = 1 << 18
    for value in (0.3, 1.7e-3, 3e-6):
        p, g = torch.zeros(n, device="cuda"), torch.full((n,), value, device="cuda")
        g[::32] = 1.0
        state = eng.adamW_state([p], 8)
        eng.adamW([p], [g], state, 1, LR, B1, B2, EPS, 0.0, seed=3)
        keep = torch.ones(n, dtype=torch.bool, device="cuda")
        keep[::32] = False
        for codes, scales, want in ((state.m[0], state.m_scale[0], (1 - B1) * value), (state.v[0], state.v_scale[0], (1 - B2) * value * value)):
            got, unit = decode(codes, scales)[keep].double(), float(scales.float()[0])
            step = max(2.0 ** -9, 2.0 ** math.floor(math.log2(want / unit)) / 8) * unit
            if codes is state.v[0] and want < step:
                assert (got >= step).all()
            else:
                assert abs(float(got.mean()) - want) <= 5 * 0.5 * step / keep.sum().item() ** 0.5 + 1e-6 * want
    # successive steps and seeds draw other bits
    p, g = torch.zeros(4096, device="cuda"), torch.full((4096,), 0.3, device="cuda")
    g[::32] = 1.0
    seen = []
    for step, seed in ((1, 0), (2, 0), (1, 1)):
        state = eng.adamW_state([p], 8)
        eng.adamW([p], [g], state, step, LR, seed=seed)
        seen.append(state.m[0].float())
    assert all(0.2 < float((a != b).float().mean()) < 0.8 for a, b in ((seen[0], seen[1]), (seen[0], seen[2]), (seen[1], seen[2])))


def test_moments_fall(eng):
    """Without gradients v falls by b2 a step: after 1000 steps its mean is e^-1 of what it was (rounded to nearest it would stand still)."""
    n = 1 << 16
    gen = torch.Generator(device="cuda").manual_seed(2)
    p, g = torch.zeros(n, device="cuda"), normal(gen, n, 1.0)
    state = eng.adamW_state([p], 8)
    eng.adamW([p], [g], state, 1, 0.0)
    first = float(decode(state.v[0], state.v_scale[0]).mean())
    g.zero_()
    for step in range(2, 1002):
        eng.adamW([p], [g], state, step, 0.0)
    # (2048 blocks whose largest element each rounds by 6 % or less a few times: well within 10 % of the mean)
    assert abs(float(decode(state.v[0], state.v_scale[0]).mean()) / first - B2 ** 1000) < 0.1 * B2 ** 1000


@pytest.mark.parametrize("bits", (32, 8))
def test_clipped_in_the_same_pass(eng, bits):
    gen = torch.Generator(device="cuda").manual_seed(3)
    params = [normal(gen, n, 0.1) for n in (5000, 33, 70000)]
    grads = [normal(gen, p.numel(), 1.0, torch.bfloat16) for p in params]
    ref = math.sqrt(sum(float((g.double() ** 2).sum()) for g in grads))
    for max_norm in (0.3 * ref, 2 * ref):
        before, state = [p.clone() for p in params], eng.adamW_state(params, bits)
        norm = eng.adamW(params, grads, state, 1, LR, B1, B2, EPS, WD, max_norm=max_norm)
        assert abs(float(norm) - ref) <= 5 * E * ref
        for p0, p1, g in zip(before, params, grads):
            check_step(p0, g, torch.zeros(g.numel(), dtype=torch.float64, device="cuda"), torch.zeros(g.numel(), dtype=torch.float64, device="cuda"), p1, 1, c=min(1.0, max_norm / (ref + 1e-6)), clipped=8)
        # the norm may come from elsewhere
        again, other = [p.clone() for p in before], eng.adamW_state(params, bits)
        assert eng.adamW(again, grads, other, 1, LR, B1, B2, EPS, WD, max_norm=max_norm, norm=norm) is norm
        assert all(torch.equal(a, b) for a, b in zip(again, params))
    for bad in (float("inf"), float("nan")):
        grads[1][5] = bad
        held = [t.clone() for t in params + state.m + state.v]
        norm = eng.adamW(params, grads, state, 2, LR, max_norm=1.0)
        assert not math.isfinite(float(norm)) and all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(held, params + state.m + state.v))


def test_missing_gradients_and_numbers(eng):
    """A tensor without a gradient is left as it is, and the others' random bits do not change for it."""
    gen = torch.Generator(device="cuda").manual_seed(4)
    params = [normal(gen, 5000, 0.1) for _ in range(3)]
    grads = [normal(gen, 5000, 1.0) for _ in range(3)]
    all_of, some = [p.clone() for p in params], [p.clone() for p in params]
    a, b = eng.adamW_state(params, 8), eng.adamW_state(params, 8)
    eng.adamW(all_of, grads, a, 1, LR)
    eng.adamW(some, [grads[0], None, grads[2]], b, 1, LR)
    assert torch.equal(some[1], params[1]) and torch.equal(some[2], all_of[2]) and torch.equal(a.m[2].view(torch.uint8), b.m[2].view(torch.uint8)) and not b.m[1].view(torch.uint8).any()
    assert eng.adamW([params[0]], [None], eng.adamW_state(params[:1]), 1, LR) is None
    assert float(eng.adamW([], [], eng.adamW_state([]), 1, LR, max_norm=1.0)) == 0.0


@pytest.mark.parametrize("bits", (32, 8))
def test_any_alignment(eng, bits):
    """Views that start anywhere: the same bits as dense tensors."""
    gen = torch.Generator(device="cuda").manual_seed(5)
    n = 9001
    p, g = normal(gen, n, 0.1, torch.bfloat16), normal(gen, n, 1.0, torch.bfloat16)
    want, state = p.clone(), eng.adamW_state([p], bits)
    eng.adamW([want], [g], state, 1, LR)
    for off in (1, 2, 3):
        view = lambda t: torch.cat([t.new_zeros(off), t.reshape(-1)])[off:]      # noqa: E731
        again, mine = view(p), eng.adamW_state([p], bits)
        mine.m, mine.v = [view(mine.m[0].view(torch.uint8)).view(mine.m[0].dtype)] if bits == 8 else [view(mine.m[0])], [view(mine.v[0].view(torch.uint8)).view(mine.v[0].dtype)] if bits == 8 else [view(mine.v[0])]
        eng.adamW([again], [view(g)], mine, 1, LR)
        assert torch.equal(again, want) and torch.equal(mine.m[0].view(torch.uint8), state.m[0].view(torch.uint8)) and torch.equal(mine.v[0].view(torch.uint8), state.v[0].view(torch.uint8))
    stepped = torch.stack([g, g], 1)[:, 0]
    again, mine = p.clone(), eng.adamW_state([p], bits)
    eng.adamW([again], [stepped], mine, 1, LR)
    assert not stepped.is_contiguous() and torch.equal(again, want)


@pytest.mark.parametrize("bits", (32, 8))
def test_capture_and_replay(eng, bits):
    """A captured step whose step number, rate and gradients change between replays, beside the same steps taken eagerly."""
    gen = torch.Generator(device="cuda").manual_seed(6)
    params = [normal(gen, n, 0.1) for n in (5000, 4097)]
    grads = [torch.zeros_like(p) for p in params]
    mine, state, other = [p.clone() for p in params], eng.adamW_state(params, bits), eng.adamW_state(params, bits)
    step, lr = torch.zeros((), dtype=torch.int64, device="cuda"), torch.zeros((), device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        eng.grad_norm(grads)                     # (its scratch)
        with torch.cuda.graph(graph, stream=s):
            step += 1
            eng.adamW(mine, grads, state, step, lr, max_norm=1.0)
    for i in range(1, 4):
        for g in grads:
            g.copy_(normal(gen, g.numel(), 1.0))
        lr.fill_(LR / i)
        graph.replay()
        eng.adamW(params, grads, other, i, float(lr), max_norm=1.0)
        torch.cuda.synchronize()
        # (size and root are formed in 64 bits on either side, by two libraries' powers)
        assert all(torch.allclose(a, b, rtol=4 * E, atol=1e-9) for a, b in zip(mine, params))
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(state.m + state.v, other.m + other.v))


def test_other_streams(eng, pkg):
    gen = torch.Generator(device="cuda").manual_seed(7)
    p, g = normal(gen, 100000, 0.1), normal(gen, 100000, 1.0)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    own = pkg.submodule("engine").Engine(pkg.submodule("engine").CudaFloat32EngineBase(stream=s))
    a, b = p.clone(), p.clone()
    torch.cuda.synchronize()
    own.adamW([a], [g], own.adamW_state([a]), 1, LR, max_norm=1.0)
    s.synchronize()
    eng.adamW([b], [g], eng.adamW_state([b]), 1, LR, max_norm=1.0)
    assert torch.equal(a, b)


def test_refusals(eng, lib, pkg):
    State = pkg.submodule("engine").AdamWState
    p, g = torch.zeros(64, device="cuda"), torch.zeros(64, device="cuda")
    state, eight = eng.adamW_state([p]), eng.adamW_state([p], 8)
    for bad in (lambda: eng.adamW([p], [], state, 1, LR), lambda: eng.adamW([p], [g], state, 1, LR, weight_decay=[0.1, 0.2]), lambda: eng.adamW([p], [g.double()], state, 1, LR),
                lambda: eng.adamW([p[::2]], [g[::2]], eng.adamW_state([p[:32]]), 1, LR), lambda: eng.adamW([p], [g[:32]], state, 1, LR), lambda: eng.adamW([p], [g.cpu()], state, 1, LR),
                lambda: eng.adamW([p[:32]], [g[:32]], state, 1, LR), lambda: eng.adamW([p], [g], state, 1, LR, norm=g[0]), lambda: eng.adamW([p], [g], state, 1, LR, seed=-1),
                lambda: eng.adamW([p], [g], state, 1, LR, seed=2 ** 32), lambda: eng.adamW([p], [g], state, torch.ones((), device="cuda"), LR), lambda: eng.adamW_state([p], 16),
                lambda: eng.adamW([p], [g], state, 1, torch.ones((), dtype=torch.float64, device="cuda")), lambda: eng.adamW([p], [g], state, 1, LR, max_norm=1.0, norm=1.0),
                lambda: State(state.m, eight.v), lambda: State(eight.m, eight.v, eight.m_scale), lambda: State(eight.m, eight.v, eight.m_scale, [s[:1] for s in eight.v_scale]),
                lambda: State(state.m, []), lambda: State([p.view(8, 8).t()], [p.view(8, 8).t()])):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: eng.adamW([p], [g], state, 0, LR), lambda: eng.adamW([p], [g], state, 1, -1.0), lambda: eng.adamW([p], [g], state, 1, LR, beta1=1.0), lambda: eng.adamW([p], [g], state, 1, LR, eps=-1.0),
                lambda: eng.adamW([p], [p], state, 1, LR), lambda: eng.adamW([p], [g], state, 1, LR, Out=[p]), lambda: eng.adamW([p, p], [g, g], eng.adamW_state([p, p]), 1, LR),
                lambda: eng.adamW([p], [g], State([p], state.v), 1, LR), lambda: eng.adamW([p], [g], state, 1, LR, max_norm=-1.0), lambda: eng.adamW([p], [g], state, 1, LR, weight_decay=-0.1)):
        with pytest.raises(lib.AlphaConvError) as e:
            bad()
        assert e.value.code == -1
