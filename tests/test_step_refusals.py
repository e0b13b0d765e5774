"""What group normalisation, the softmax cross entropy of a FullConnect layer and AdamW refuse, at the C ABI: every check comes before the device is looked at."""
import ctypes as C

import pytest


@pytest.fixture(scope="module")
def lib(pkg):
    return pkg.submodule("lib")


def at(i):
    return i << 36


def refused(lib, rc, word):
    assert rc == -1 and word in lib.last_error(), (rc, lib.last_error())


NAN, INF = float("nan"), float("inf")


def norm(lib, back=False, N=2, positions=64, C_=32, groups=4, dtype=1, affine=1, act=3, k=0.0, eps=1e-5, x=at(1), gamma=at(2), beta=at(3), mean=at(4), rstd=at(5), y=at(6), dy=at(7), dg=at(8), db=at(9)):
    s, L = lib.AlphaNormShape(N, positions, C_, groups, dtype, affine, act, k, eps), lib.load()
    if back:
        return L.alpha_groupNorm_delta(C.byref(s), dy, x, mean, rstd, gamma, beta, y, dg, db, None)
    return L.alpha_groupNorm(C.byref(s), x, gamma, beta, mean, rstd, y, None)


@pytest.mark.parametrize("back", (False, True))
@pytest.mark.parametrize("kw,word", [
    (dict(N=0), "non-positive"), (dict(positions=-1), "non-positive"), (dict(C_=0), "non-positive"), (dict(groups=0), "non-positive"), (dict(groups=5), "groups of one size"),
    (dict(positions=2 ** 31 - 1), "more than"), (dict(N=2 ** 27), "more than"), (dict(dtype=3), "element type"), (dict(affine=2), "fp32"), (dict(dtype=0, affine=1), "fp32"),
    (dict(act=6), "activation"), (dict(act=1, k=NAN), "slope"), (dict(eps=-1.0), "eps"), (dict(eps=NAN), "eps"), (dict(eps=INF), "eps"),
    (dict(x=None), "null"), (dict(y=None), "null"), (dict(beta=None), "null"), (dict(gamma=None), "null"), (dict(rstd=None), "null"),
    (dict(x=at(1) + 1), "aligned"), (dict(y=at(6) + 1), "aligned"), (dict(mean=at(4) + 2), "aligned"), (dict(gamma=at(2) + 1), "aligned"),
    (dict(y=at(1)), "overlaps"), (dict(y=at(1) + 2 * 64 * 32 * 2 - 2), "overlaps"), (dict(y=at(2) - 4), "overlap"),
])
def test_group_norm(lib, back, kw, word):
    refused(lib, norm(lib, back, **kw), word)


@pytest.mark.parametrize("kw,word", [(dict(mean=None, rstd=None), "null"), (dict(dy=None), "null"), (dict(dg=None), "null"), (dict(db=None), "null"), (dict(y=at(7)), "overlaps"), (dict(dg=at(9)), "overlap"),
                                     (dict(dg=at(3)), "overlaps"), (dict(db=at(9) + 1), "aligned")])
def test_group_norm_gradients(lib, kw, word):
    refused(lib, norm(lib, True, **kw), word)


def test_group_norm_moments_apart(lib):
    refused(lib, norm(lib, mean=at(4), rstd=at(4) + 4), "overlap")
    refused(lib, norm(lib, mean=at(6)), "overlap")


def loss(lib, back=False, rows=16, IC=64, OC=40, dtype=1, act=0, x=at(1), w=at(2), b=None, label=at(3), size=8, out=at(4), lse=at(5), dl=at(6), step=1, dx=at(7), dw=at(8), db=at(9)):
    s, L = lib.AlphaFcShape(rows, IC, OC, dtype, act, 0.0), lib.load()
    if back:
        return L.alpha_fullConnect_softmax_crossEntropy_delta(C.byref(s), dl, step, x, w, b, label, size, lse, dx, dw, db, None)
    return L.alpha_fullConnect_softmax_crossEntropy(C.byref(s), x, w, b, label, size, out, lse, None)


@pytest.mark.parametrize("back", (False, True))
@pytest.mark.parametrize("kw,word", [
    (dict(rows=0), "non-positive"), (dict(IC=0), "non-positive"), (dict(OC=-3), "non-positive"), (dict(IC=60), "multiple of 8"), (dict(IC=62, dtype=0), "multiple of 4"), (dict(dtype=4), "element type"),
    (dict(act=3), "no activation"), (dict(label=None), "labels"), (dict(size=2), "labels"), (dict(label=at(3) + 4), "labels"), (dict(size=4, label=at(3) + 2), "labels"),
    (dict(x=None), "null"), (dict(w=None), "null"), (dict(x=at(1) + 8), "aligned"), (dict(w=at(2) + 2), "aligned"), (dict(b=at(10) + 8), "aligned"), (dict(lse=at(5) + 2), "floats"),
    (dict(rows=1 << 20, IC=4096, dtype=0), "2^31-1"), (dict(rows=1 << 20, OC=4096, dtype=0), "2^31-1"), (dict(OC=2 ** 31 - 1), "dimension"),
])
def test_loss(lib, back, kw, word):
    refused(lib, loss(lib, back, **kw), word)


@pytest.mark.parametrize("kw,word", [(dict(out=None, lse=None), "null"), (dict(out=at(5)), "overlap"), (dict(out=at(1) + 4), "overlaps"), (dict(lse=at(3)), "overlaps"), (dict(out=at(4) + 1), "floats")])
def test_loss_outputs(lib, kw, word):
    refused(lib, loss(lib, **kw), word)


@pytest.mark.parametrize("kw,word", [(dict(lse=None), "null"), (dict(dl=None), "null"), (dict(step=2), "step"), (dict(dx=None, dw=None, db=None), "no gradient"), (dict(dx=at(1)), "overlaps"), (dict(dw=at(2)), "overlaps"),
                                     (dict(dx=at(8)), "overlap"), (dict(dx=at(5)), "overlaps"), (dict(dw=at(3)), "overlaps"), (dict(dx=at(6)), "overlaps"), (dict(dx=at(7) + 8), "aligned"), (dict(dl=at(6) + 2), "floats")])
def test_loss_gradients(lib, kw, word):
    refused(lib, loss(lib, True, **kw), word)


def adam(lib, rows=None, n=None, step=1, lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, max_norm=0.0, norm=None, lr_at=None, step_at=None, **kw):
    if rows is None:
        rows = [dict(kw)]
    full = dict(param=at(1), grad=at(2), m=at(3), v=at(4), m_scale=None, v_scale=None, out=None, count=100, weight_decay=0.0, dtype=0, grad_dtype=0, out_dtype=0, moment_bits=32)
    table = (lib.AlphaAdamW * len(rows))(*[lib.AlphaAdamW(**{**full, **r}) for r in rows])
    how = lib.AlphaAdamWStep(lr, beta1, beta2, eps, max_norm, step, norm, lr_at, step_at, 0)
    return lib.load().alpha_adamW(len(rows) if n is None else n, C.cast(table, C.c_void_p), C.byref(how), None)


@pytest.mark.parametrize("kw,word", [
    (dict(n=-1), "null"), (dict(step=0), "step"), (dict(step=-5), "step"), (dict(lr=-1.0), "lr"), (dict(lr=NAN), "lr"), (dict(lr=INF), "lr"), (dict(beta1=1.0), "beta1"), (dict(beta2=-0.1), "beta2"), (dict(beta2=NAN), "beta2"),
    (dict(eps=-1e-8), "eps"), (dict(eps=INF), "eps"), (dict(norm=at(9), max_norm=NAN), "max_norm"), (dict(norm=at(9), max_norm=-1.0), "max_norm"), (dict(norm=at(9) + 2), "aligned"),
    (dict(lr_at=at(9) + 1), "aligned"), (dict(step_at=at(9) + 4), "aligned"), (dict(dtype=3), "element type"), (dict(grad_dtype=-1), "element type"), (dict(out=at(5), out_dtype=9), "element type"),
    (dict(moment_bits=16), "bits"), (dict(count=-1), "elements"), (dict(count=1 << 42), "elements"), (dict(weight_decay=-0.1), "decay"), (dict(weight_decay=NAN), "decay"),
    (dict(param=None), "null"), (dict(grad=None), "null"), (dict(m=None), "null"), (dict(v=None), "null"), (dict(moment_bits=8), "null"), (dict(moment_bits=8, m_scale=at(6)), "null"),
    (dict(param=at(1) + 2), "aligned"), (dict(grad=at(2) + 1, grad_dtype=1), "aligned"), (dict(v=at(4) + 2), "aligned"), (dict(out=at(5) + 2), "aligned"),
    (dict(grad=at(1)), "overlaps"), (dict(m=at(4) + 396), "overlaps"), (dict(out=at(1)), "overlaps"), (dict(out=at(2) + 396), "overlaps"), (dict(norm=at(1) + 4), "overlaps"), (dict(step_at=at(3)), "overlaps"),
    (dict(moment_bits=8, m_scale=at(6), v_scale=at(6) + 3), "overlaps"), (dict(moment_bits=8, m=at(3), v=at(3) + 99, m_scale=at(6), v_scale=at(7)), "overlaps"),
])
def test_adamw(lib, kw, word):
    refused(lib, adam(lib, **kw), word)


def test_adamw_tensors_together(lib):
    second = dict(param=at(11), grad=at(12), m=at(13), v=at(14))
    refused(lib, adam(lib, rows=[{}, {**second, "grad": at(1)}]), "overlaps")
    refused(lib, adam(lib, rows=[{}, {**second, "m": at(3)}]), "overlaps")
    refused(lib, adam(lib, rows=[{}, {**second, "moment_bits": 8, "m_scale": at(15), "v_scale": at(16)}]), "all 8")
    refused(lib, lib.load().alpha_adamW(1, None, C.byref(lib.AlphaAdamWStep()), None), "null")
    refused(lib, lib.load().alpha_adamW(0, None, None, None), "null")


def test_sizes_of_structures(lib):
    """The table the Python calls pack is the header's structure."""
    import struct
    assert C.sizeof(lib.AlphaAdamW) == struct.calcsize("@7Pqd4i") == 88 and C.sizeof(lib.AlphaNormShape) == 36 and C.sizeof(lib.AlphaAdamWStep) == 80


def test_workspace_arguments(lib):
    n = C.c_size_t(0)
    refused(lib, lib.load().alpha_groupNorm_workspace_bytes(None, 0, C.byref(n)), "null")
    refused(lib, lib.load().alpha_groupNorm_workspace_bytes(C.byref(lib.AlphaNormShape(1, 1, 4, 1, 0, 0, 0, 0.0, 0.0)), 2, C.byref(n)), "unknown op")
    refused(lib, lib.load().alpha_fullConnect_softmax_crossEntropy_workspace_bytes(None, 0, C.byref(n)), "null")
    refused(lib, lib.load().alpha_fullConnect_softmax_crossEntropy_workspace_bytes(C.byref(lib.AlphaFcShape(1, 8, 4, 1, 0, 0.0)), 3, C.byref(n)), "unknown op")


def test_states_without_a_gpu(pkg):
    """The moments' checks need no GPU."""
    torch = pytest.importorskip("torch")
    E = pkg.submodule("engine")
    p = [torch.zeros(5, 7), torch.zeros(64)]
    for bits in (32, 8):
        s = E.Engine.adamW_state(p, bits)
        assert s.bits == bits and [m.shape for m in s.m] == [t.shape for t in p]
    assert [t.numel() for t in s.m_scale] == [2, 2] and s.m[0].dtype == torch.float8_e4m3fn and s.v_scale[0].dtype == torch.float8_e8m0fnu
    for bad in (lambda: E.Engine.adamW_state(p, 4), lambda: E.AdamWState(s.m, s.v), lambda: E.AdamWState(s.m, s.v, s.m_scale), lambda: E.AdamWState(s.m, s.v[:1], s.m_scale, s.v_scale),
                lambda: E.AdamWState([t.double() for t in p], p)):
        with pytest.raises(ValueError):
            bad()
