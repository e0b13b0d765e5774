"""The cache of FullConnect shapes sees plain ints: what no size is, is refused whether or not an equal size was used before; a size that changes is read anew."""
import pytest

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def engine(pkg):
    return pkg.submodule("engine")


CALLS = {
    "fullConnect": lambda b, rows, IC, OC, dtype, act, k: b.fullConnect(7 << 32, 1 << 32, 2 << 32, rows, IC, OC, dtype, act, k),
    "fullConnect_glu": lambda b, rows, IC, OC, dtype, act, k: b.fullConnect_glu(7 << 32, 1 << 32, 2 << 32, rows, IC, OC, dtype, act, k),
    "fullConnect_delta": lambda b, rows, IC, OC, dtype, act, k: b.fullConnect_delta(7 << 32, 8 << 32, None, 3 << 32, 1 << 32, 2 << 32, 4 << 32, 4 << 32, rows, IC, OC, dtype, act, k),
}


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("at", range(5))
@pytest.mark.parametrize("seen", (False, True))
def test_sizes_are_whole_numbers(engine, name, at, seen):
    base = engine.CudaFloat32EngineBase()
    args = [16, 24, 40, 1, 3, 0.0]
    engine._cached_fc_shape.cache_clear()
    if seen:
        engine._cached_fc_shape(*args)
    args[at] = float(args[at])
    with pytest.raises(TypeError, match="integer"):
        CALLS[name](base, *args)


def test_a_tensor_is_read_when_it_is_given(engine):
    rows = torch.tensor(16)
    assert engine._fc_shape(rows, 24, 40, 1, 3, 0).rows == 16
    rows.fill_(5)
    assert engine._fc_shape(rows, 24, 40, 1, 3, 0).rows == 5
    k = torch.tensor(0.5)
    assert engine._fc_shape(5, 24, 40, 1, 1, k).k == 0.5
    k.fill_(0.25)
    assert engine._fc_shape(5, 24, 40, 1, 1, k).k == 0.25
