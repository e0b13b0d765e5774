"""What fullConnect, its gradients and clip_grad_norm refuse, at the C ABI: every check comes before the device is looked at."""
import ctypes as C
import struct

import pytest


@pytest.fixture(scope="module")
def lib(pkg):
    return pkg.submodule("lib")


X, W, B, R, Z, Y, D = (i << 32 for i in range(1, 8))
BF16 = 1


def refused(lib, rc, word):
    assert rc == -1 and word in lib.last_error(), (rc, lib.last_error())


def call(lib, rows=16, IC=64, OC=32, dtype=BF16, act=0, k=0.0, x=X, w=W, b=None, r=None, z=None, y=Y, glu=False):
    s = lib.AlphaFcShape(rows, IC, OC, dtype, act, k)
    L = lib.load()
    return L.alpha_fullConnect_glu(C.byref(s), x, w, b, z, y, None) if glu else L.alpha_fullConnect(C.byref(s), x, w, b, r, z, y, None)


@pytest.mark.parametrize("glu", (False, True))
@pytest.mark.parametrize("kw,word", [
    (dict(rows=0), "non-positive"), (dict(rows=-1), "non-positive"), (dict(IC=0), "non-positive"), (dict(OC=0), "non-positive"),
    (dict(IC=60), "multiple of 8"), (dict(IC=62, dtype=0), "multiple of 4"),
    (dict(dtype=3), "element type"), (dict(dtype=-1), "element type"), (dict(act=6), "activation"), (dict(act=-1), "activation"),
    (dict(act=1, k=float("nan")), "slope"), (dict(x=None), "null"), (dict(w=None), "null"), (dict(y=None), "null"),
    (dict(x=X + 8), "aligned"), (dict(w=W + 2), "aligned"), (dict(y=Y + 4), "aligned"), (dict(b=B + 8), "aligned"), (dict(z=Z + 8), "aligned"),
    (dict(y=X), "overlaps"), (dict(y=X + 16 * 64 * 2 - 16), "overlaps"), (dict(z=W), "overlaps"), (dict(z=Y), "overlap"), (dict(b=Y), "overlaps"),
    (dict(rows=2 ** 31 - 1023), "dimension"), (dict(IC=2 ** 31 - 8), "dimension"), (dict(OC=2 ** 31 - 1), "dimension"),
    (dict(rows=1 << 20, IC=4096, dtype=0), "2^31-1"), (dict(rows=1 << 20, OC=4096, dtype=0), "2^31-1"),
])
def test_forward(lib, glu, kw, word):
    refused(lib, call(lib, glu=glu, **kw), word)


def test_residual(lib):
    refused(lib, call(lib, r=Y + 16), "overlaps")
    refused(lib, call(lib, r=R + 8), "aligned")
    refused(lib, call(lib, r=Z, z=Z), "overlaps")


def delta(lib, rows=16, IC=64, OC=32, dtype=BF16, act=3, dy=Y, x=X, w=W, z=Z, dz=D, dx=8 << 32, dw=9 << 32, db=10 << 32, glu=False):
    s = lib.AlphaFcShape(rows, IC, OC, dtype, act, 0.0)
    fn = lib.load().alpha_fullConnect_glu_delta if glu else lib.load().alpha_fullConnect_delta
    return fn(C.byref(s), dy, x, w, z, dz, dx, dw, db, None)


@pytest.mark.parametrize("glu", (False, True))
@pytest.mark.parametrize("kw,word", [
    (dict(rows=0), "non-positive"), (dict(dtype=7), "element type"), (dict(act=9), "activation"), (dict(IC=33), "multiple"),
    (dict(dy=None), "null"), (dict(x=None), "null"), (dict(w=None), "null"), (dict(z=None), "Z of the forward pass"), (dict(dz=None), "Z of the forward pass"),
    (dict(dx=None, dw=None, db=None), "no gradient"), (dict(dz=Y), "overlaps"), (dict(dz=Z + 16), "overlaps"), (dict(dx=X), "overlaps"), (dict(dw=W), "overlaps"),
    (dict(dx=Z), "overlap"), (dict(db=9 << 32), "overlap"), (dict(dx=(8 << 32) + 8), "aligned"), (dict(db=(10 << 32) + 2), "aligned"),
])
def test_delta(lib, glu, kw, word):
    refused(lib, delta(lib, glu=glu, **kw), word)


def test_workspace_arguments(lib):
    s, n = lib.AlphaFcShape(16, 64, 32, BF16, 0, 0.0), C.c_size_t(0)
    refused(lib, lib.load().alpha_fullConnect_workspace_bytes(None, 0, 0, C.byref(n)), "null")
    refused(lib, lib.load().alpha_fullConnect_workspace_bytes(C.byref(s), 0, 2, C.byref(n)), "unknown op")


def clip(lib, entries, max_norm=1.0, norm=20 << 32, scale=True):
    t = (lib.AlphaGrad * max(len(entries), 1))(*[lib.AlphaGrad(*e) for e in entries])
    L = lib.load()
    return L.alpha_clip_grad_norm(len(entries), t, max_norm, norm, None) if scale else L.alpha_grad_norm(len(entries), t, norm, None)


@pytest.mark.parametrize("entries,word", [
    ([(X, X, -1, 0, 0)], "elements"), ([(X, X, 1 << 60, 0, 0)], "elements"), ([(None, X, 4, 0, 0)], "null"), ([(X, None, 4, 0, 0)], "null"),
    ([(X, X, 4, 5, 0)], "element type"), ([(X, X, 4, 0, 3)], "element type"), ([(X + 2, X + 2, 4, 0, 0)], "aligned"), ([(X + 1, Y, 4, 1, 0)], "aligned"),
    ([(X, Y + 1, 4, 0, 1)], "aligned"), ([(X, X, 4, 0, 1)], "overlaps"), ([(X, X + 4, 4, 0, 0)], "overlaps"), ([(X, X, 8, 0, 0), (X, X, 8, 0, 0)], "overlaps"),
    ([(X, X, 8, 0, 0), (X + 16, Y, 8, 0, 0)], "overlaps"), ([(X, Y, 8, 0, 0), (W, Y + 28, 8, 0, 0)], "overlaps"), ([(20 << 32, X, 1, 0, 0)], "overlaps"),
])
def test_clip(lib, entries, word):
    refused(lib, clip(lib, entries), word)


def test_clip_arguments(lib):
    ok = [(X, X, 4, 0, 0)]
    for bad in (-1.0, float("nan")):
        refused(lib, clip(lib, ok, max_norm=bad), "max_norm")
    for bad in (None, (20 << 32) + 2):
        refused(lib, clip(lib, ok, norm=bad), "norm must be")
        refused(lib, clip(lib, ok, norm=bad, scale=False), "norm must be")
    refused(lib, lib.load().alpha_grad_norm(2, None, 20 << 32, None), "no tensors")
    refused(lib, lib.load().alpha_grad_norm(-1, None, 20 << 32, None), "no tensors")


# ---- Engine: shapes, types and devices, before anything is launched (tensors of the meta and the CPU device) ----

@pytest.fixture(scope="module")
def eng(pkg):
    return pkg.submodule("engine").Engine()


def _t(*shape, dtype=None):
    torch = pytest.importorskip("torch")
    return torch.zeros(shape, dtype=dtype or torch.float32)


@pytest.mark.parametrize("glu", (False, True))
def test_engine_forward(eng, glu):
    torch = pytest.importorskip("torch")
    fn = eng.fullConnect_glu if glu else eng.fullConnect
    for args, kw, word in [
        ((_t(4, 8), _t(6, 9)), {}, "against W"), ((_t(4, 8), _t(6, 8, 1)), {}, "against W"), ((_t(4, 0), _t(6, 0)), {}, "against W"), ((_t(4, 8), _t(0, 8)), {}, "against W"),
        ((_t(4, 8, dtype=torch.float64), _t(6, 8, dtype=torch.float64)), {}, "float32, bfloat16 or float16"), ((_t(4, 8), _t(6, 8)), dict(act="relu"), "act must be one of"),
        ((_t(4, 8), _t(6, 8)), {}, "on a GPU"),
    ]:
        with pytest.raises(ValueError, match=word):
            fn(*args, **kw)
    if glu:
        with pytest.raises(ValueError, match="gate rows and as many up rows"):
            fn(_t(4, 8), _t(7, 8))


def test_engine_grads(eng):
    with pytest.raises(ValueError, match="1 gradients, 2 outputs"):
        eng.clip_grad_norm([_t(4)], 1.0, Out=[_t(4), _t(4)])
    with pytest.raises(ValueError, match="on one GPU"):
        eng.clip_grad_norm([_t(4)], 1.0)
    with pytest.raises(ValueError, match="on one GPU"):
        eng.grad_norm([_t(4)])


@pytest.mark.parametrize("glu", (False, True))
def test_engine_sizes_past_an_int(eng, glu):
    torch = pytest.importorskip("torch")
    t = lambda *shape: torch.empty(shape, dtype=torch.bfloat16, device="meta")
    for x, w in ((t(2 ** 31, 8), t(16, 8)), (t(2 ** 16, 2 ** 15, 8), t(16, 8)), (t(2, 2 ** 31), t(16, 2 ** 31)), (t(2, 8), t(2 ** 32, 8))):
        with pytest.raises(ValueError, match="too large"):
            (eng.fullConnect_glu if glu else eng.fullConnect)(x, w)


@pytest.mark.parametrize("job,dtype,word", [
    ((X, 3, 5, Y, 3, 8), 3, "element type"), ((X, 3, 5, Y, 3, 8), -1, "element type"), ((0, 3, 5, Y, 3, 8), 1, "null"), ((X, 3, 5, 0, 3, 8), 1, "null"),
    ((X, 0, 5, Y, 3, 8), 1, "bad shape"), ((X, 3, 0, Y, 3, 8), 1, "bad shape"), ((X, 3, 5, Y, 2, 8), 1, "bad shape"), ((X, 3, 9, Y, 3, 8), 1, "bad shape"),
    ((X, 3, 5, Y, 3, 12), 1, "bad shape"), ((X, 3, 5, Y, 3, 6), 0, "bad shape"), ((X, 3, 5, Y, 3, 1 << 31), 1, "bad shape"),
    ((X + 1, 3, 5, Y, 3, 8), 1, "aligned"), ((X + 2, 3, 5, Y, 3, 8), 0, "aligned"), ((X, 3, 5, Y + 8, 3, 8), 1, "aligned"),
])
def test_pad_rows_typed(lib, job, dtype, word):
    refused(lib, lib.load().alpha_pad_rows_typed(1, struct.pack("6q", *job), dtype, None), word)
    refused(lib, lib.load().alpha_pad_rows_typed(2, struct.pack("12q", X, 1, 8, Z, 1, 8, *job), dtype, None), word)
    refused(lib, lib.load().alpha_pad_rows_typed(0, b"", 1, None), "no jobs")
