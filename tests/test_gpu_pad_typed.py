"""alpha_pad_rows_typed: zero-padded copies of many tensors of one type, eight to a launch, bit for bit."""
import struct

import pytest

pytestmark = pytest.mark.gpu

# rows, cols, rows4, cols4: a single element, sources that start anywhere, more rows than the source's, whole words, longer rows than needed
SHAPES = [(1, 1, 1, 8), (7, 3, 8, 8), (300, 5, 300, 8), (13, 257, 16, 264), (70000, 3, 70000, 8), (5, 16, 5, 16), (2, 9, 2, 48), (1000, 1001, 1000, 1008), (3, 8, 5, 8), (64, 31, 64, 32)]


def pad(pkg, jobs, dtype):
    import torch
    lib = pkg.submodule("lib")
    values = [v for src, rows, cols, out, rows4, cols4 in jobs for v in (src.data_ptr(), rows, cols, out.data_ptr(), rows4, cols4)]
    lib.check(lib.load().alpha_pad_rows_typed(len(jobs), struct.pack("%dq" % len(values), *values), {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[dtype],
                                              torch.cuda.current_stream().cuda_stream))


@pytest.mark.parametrize("dtype", ("float32", "bfloat16", "float16"))
@pytest.mark.parametrize("most", (1, 8, 10))
def test_many(pkg, dtype, most):
    import torch
    dtype = getattr(torch, dtype)
    bits = torch.int32 if dtype == torch.float32 else torch.int16
    jobs, wants = [], []
    for i, (rows, cols, rows4, cols4) in enumerate(SHAPES[:most]):
        src = torch.randint(-30000, 30000, (rows * cols + i % 3,), device="cuda", dtype=bits)[i % 3:].view(rows, cols)      # (any bit pattern, any start)
        out = torch.full((rows4 * cols4 + 16,), 77, device="cuda", dtype=bits)
        want = torch.zeros((rows4, cols4), device="cuda", dtype=bits)
        want[:rows, :cols] = src
        jobs.append((src, rows, cols, out, rows4, cols4))
        wants.append(want)
    pad(pkg, jobs, dtype)
    for (_, rows, cols, out, rows4, cols4), want in zip(jobs, wants):
        assert torch.equal(out[:rows4 * cols4].view(rows4, cols4), want), (rows, cols)
        assert bool((out[rows4 * cols4:] == 77).all()), (rows, cols)


def test_more_words_than_a_launch_indexes(pkg):
    import torch
    rows = 2010000000
    src = torch.arange(rows, device="cuda", dtype=torch.int32).to(torch.int16)
    out = torch.full((rows + 3, 8), 77, device="cuda", dtype=torch.int16)
    pad(pkg, [(src, rows, 1, out, rows + 2, 8)], torch.bfloat16)
    assert torch.equal(out[:rows, 0], src)
    words = out.view(torch.int64)                                                  # (four elements)
    assert torch.equal(words[:rows, 0], src.to(torch.int64) & 0xffff) and int(words[:rows, 1].count_nonzero()) == 0
    assert int(out[rows:rows + 2].count_nonzero()) == 0 and bool((out[rows + 2:] == 77).all())
