"""Which tensors clip_grad_norm takes for disjoint (engine._memory_of, _apart, _refuse_overlaps), against the sets of their elements, on the CPU."""
import itertools
import random

import pytest

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def engine(pkg):
    return pkg.submodule("engine")


def elements(t):
    """Byte addresses of a tensor's elements, counted as often as they occur."""
    at = [t.data_ptr()]
    for n, st in zip(t.shape, t.stride()):
        at = [a + i * st * t.element_size() for a in at for i in range(n)]
    return at


def views(rng, base):
    """Views of a small matrix: columns, rows, transposed, strided, expanded, overlapping windows."""
    flat, n, m = base.reshape(-1), base.shape[0], base.shape[1]
    c0, r0 = rng.randrange(m), rng.randrange(n)
    c1, r1 = rng.randrange(c0 + 1, m + 1), rng.randrange(r0 + 1, n + 1)
    cut = base[r0:r1, c0:c1]
    yield from (cut, cut.T, cut.unsqueeze(1), base[r0:r1], base[::2, c0:c1], cut[..., ::2], flat[r0 * m + c0:], flat[::3], base[r0].expand(3, m), flat.as_strided((4, 3), (2, 1), c0),
                flat.as_strided((2, 3, 2), (m, 2, 1), 0), base[r0:r1, c0:c1].reshape(-1)[:0], cut[0, 0])


def test_against_the_elements(engine):
    rng = random.Random(5)
    sure = told = 0
    for _ in range(300):
        dtype = rng.choice((torch.float32, torch.bfloat16))
        base = torch.zeros(rng.randrange(3, 7), rng.randrange(6, 12), dtype=dtype)
        some = list(views(rng, base)) + list(views(rng, base.view(torch.int16).view(torch.bfloat16)))
        for t in some:
            if t.numel() == 0:
                continue
            at, place = elements(t), engine._memory_of(t)
            if len(set(at)) < len(at):
                assert place is None
            if place is not None:
                assert len(set(at)) == len(at) and place[0] == min(at) and place[1] == max(at) + t.element_size()
        for a, b in itertools.combinations([t for t in some if t.numel() and engine._memory_of(t) is not None], 2):
            held = [{x + i for x in elements(t) for i in range(t.element_size())} for t in (a, b)]
            apart = engine._apart(engine._memory_of(a), engine._memory_of(b))
            assert apart == engine._apart(engine._memory_of(b), engine._memory_of(a))
            if apart:
                assert not held[0] & held[1], (a.shape, a.stride(), b.shape, b.stride())
                told += 1
            sure += not held[0] & held[1]
    assert told > 0.5 * sure                        # (what is not rows of one pitch cannot be told)


def test_columns_of_one_matrix_are_apart(engine):
    for n, m in ((1, 8), (5, 8), (40, 33)):
        base = torch.zeros(n, m)
        for c in range(1, m):
            for a, b in ((base[:, :c], base[:, c:]), (base[1:, :c], base[:-1, c:]), (base[:, :c], base[n // 2, c:])):
                if a.numel() and b.numel():
                    assert engine._apart(engine._memory_of(a), engine._memory_of(b))
            if c + 1 < m:
                assert not engine._apart(engine._memory_of(base[:, :c + 1]), engine._memory_of(base[:, c:]))


def test_refusals(engine):
    b = torch.zeros(6, 10)
    ok = [([b[:, :5], b[:, 5:]], None), ([b[:, :5]], [b[:, 5:]]), ([b.T], [torch.zeros(10, 6)]), ([b[0].expand(3, 10)], [torch.zeros(3, 10)]), ([b[:, :0]], None),
          ([b[:, :5], b[:, :5]], [torch.zeros(6, 5), torch.zeros(6, 5)])]
    for grads, out in ok:
        engine._refuse_overlaps("clip", grads, out or grads)
    bad = [([b[:, :5], b[:, 4:]], None, "overlaps"), ([b[:, :5]], [b[:, 1:6]], "overlaps"), ([b[0].expand(3, 10)], None, "share memory"), ([b[:, :5], b[:, :5]], None, "overlaps"),
           ([b[:, :5], torch.zeros(2, 2).T], [torch.zeros(6, 5), b[2:4, 1:3]], "overlaps"), ([b], [b.T.reshape(-1).as_strided((6, 10), (1, 6))], None)]
    for grads, out, word in bad:
        if word:
            with pytest.raises(ValueError, match=word):
                engine._refuse_overlaps("clip", grads, out or grads)
        else:
            engine._refuse_overlaps("clip", grads, out or grads)       # (reshape made a copy)
