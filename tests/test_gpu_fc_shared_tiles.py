"""16-bit products whose tiles are shared by clusters of 2, 4 and 8 CTAs: each case says which plan has to run, and fails if another did.

A reduction of n stages (two blocks of 64 steps each) is shared by s CTAs only where no part is empty, (s - 1) ceil(n / s) < n, and a launch has a place for every
cluster; columns of an operand that runs along its rows come in 64s."""
import pytest

torch = pytest.importorskip("torch")

from test_gpu_fc import TYPES, delta_case, forward_case, rand

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng(pkg):
    return pkg.submodule("engine").Engine()


@pytest.fixture(scope="module")
def lib(pkg):
    return pkg.submodule("lib")


@pytest.fixture
def forced(lib):
    old = []

    def force(tile):
        old.append(lib.set_option("FC_TILE", tile))
    yield force
    for o in reversed(old):
        lib.set_option("FC_TILE", o)
    assert lib.device_status() == 0, lib.last_error()


# one row tile of few rows, a ragged one, two of them; reductions of whole stages, of a block less, of a few steps more than that
FORWARD = [(20, 1024, 136), (77, 2040, 264), (200, 1992, 129), (256, 4096, 72)]


@pytest.mark.parametrize("split", (2, 4, 8))
@pytest.mark.parametrize("bn", (16, 48, 64, 112, 128, 256))
@pytest.mark.parametrize("rows,IC,OC", FORWARD)
@pytest.mark.parametrize("glu", (False, True), ids=("fc", "glu"))
@pytest.mark.parametrize("dtype", ("bf16", "f16"))
def test_forward(eng, lib, forced, dtype, glu, rows, IC, OC, bn, split):
    most = 148 // split
    tiles = -(-rows // 128) * -(-OC // (bn // 2 if glu else bn))
    if tiles > (most if split < 4 else most * 87 // 100):
        pytest.skip("more tiles than clusters at once")
    forced(1000 * split + bn)
    forward_case(eng, lib, dtype, rows, IC, OC, "silu", glu, bias=True, residual=not glu, save=True)
    assert "128x%d split=%d" % (bn, split) in lib.last_plan(), lib.last_plan()
    if bn == 64:
        forward_case(eng, lib, dtype, rows, IC, OC, "none", glu, bias=False, residual=False, save=False, seed=1)


@pytest.mark.parametrize("split", (2, 4, 8))
@pytest.mark.parametrize("bn", (64, 128, 256))
@pytest.mark.parametrize("glu", (False, True), ids=("fc", "glu"))
@pytest.mark.parametrize("dtype", ("bf16", "f16"))
def test_gradients(eng, lib, forced, dtype, glu, bn, split):
    forced(1000 * split + bn)
    t, H, code = TYPES[dtype], 2 if glu else 1, {"bf16": 1, "f16": 2}[dtype]
    for rows, IC, OC, which in ((100, 200, 1000 if glu else 2000, 0), (2000, 72, 100, 1)):       # (16 stages of deltaX, of deltaW)
        delta_case(eng, lib, dtype, rows, IC, OC, "silu", glu, bias=True)
        gen = torch.Generator(device="cuda").manual_seed(0)
        X, W, dY, Z = rand(gen, rows, IC, dtype=t), rand(gen, H * OC, IC, scale=IC ** -0.5, dtype=t), rand(gen, rows, OC, dtype=t), rand(gen, rows, H * OC, scale=2.0, dtype=t)
        want = (eng.fullConnect_glu_delta if glu else eng.fullConnect_delta)(dY, X, W, Z, act="silu")
        P = -(-OC // 8) * 8
        pad = lambda a, n: torch.nn.functional.pad(a.reshape(rows, n, OC), (0, P - OC)).contiguous()
        out = [torch.empty_like(X), torch.empty_like(W)]
        dZ = torch.empty(rows, H, P, dtype=t, device="cuda")
        eng.base.fullConnect_delta(out[0] if which == 0 else None, out[1] if which == 1 else None, None, pad(dY, 1), X if which else None, W if not which else None, pad(Z, H), dZ,
                                   rows, IC, OC, code, lib.ACTS["silu"], 0.0, glu)
        assert "128x%d split=%d" % (bn, split) in lib.last_plan(), lib.last_plan()
        assert torch.equal(out[which], want[which])


@pytest.mark.parametrize("dtype", ("bf16", "f16"))
@pytest.mark.parametrize("split", (2, 4, 8))
def test_shared_tiles_by_a_graph_and_again(eng, lib, forced, dtype, split):
    """The same bits eagerly, captured and replayed, ten times over."""
    forced(1000 * split + 64)
    gen = torch.Generator(device="cuda").manual_seed(2)
    X, W, R = rand(gen, 150, 2048, dtype=TYPES[dtype]), rand(gen, 200, 2048, scale=0.02, dtype=TYPES[dtype]), rand(gen, 150, 200, dtype=TYPES[dtype])
    want = eng.fullConnect(X, W, act="gelu", Residual=R)
    assert "split=%d" % split in lib.last_plan()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        Y = eng.fullConnect(X, W, act="gelu", Residual=R)
    for _ in range(10):
        Y.zero_()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(Y, want)
        assert torch.equal(eng.fullConnect(X, W, act="gelu", Residual=R), want)
