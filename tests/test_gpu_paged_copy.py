"""paged_copy against indexing."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from trifuse_b200 import ops as _ops
    return _ops


def filled(*shape, dtype=torch.uint8, seed=0):
    g = torch.Generator().manual_seed(seed)
    n = torch.empty(shape, dtype=dtype).element_size()
    x = torch.randint(0, 256, (*shape[:-1], shape[-1] * n), generator=g, dtype=torch.uint8)
    return x.view(dtype).cuda()


def check(ops, arrays, src, dst):
    want = []
    for t in arrays:
        w = t.contiguous().view(torch.uint8).clone()
        w[:, dst] = w[:, src]
        want.append(w)
    ops.paged_copy(arrays, src, dst)
    for t, w in zip(arrays, want):
        assert torch.equal(t.contiguous().view(torch.uint8), w)


@pytest.mark.parametrize("layers,pages,heads,page,D", [(1, 2, 1, 16, 64), (16, 40, 16, 16, 128), (3, 33, 2, 64, 64),
                                                       (2, 9, 8, 256, 128), (5, 700, 1, 16, 64)])
def test_caches(ops, layers, pages, heads, page, D):
    """16-bit keys and values; 8-bit ones with their scales: every number of pairs that fits."""
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(1)).tolist()
    for n in sorted({1, min(3, pages // 2), pages // 2}):
        src, dst = order[:n], order[n:2 * n]
        check(ops, [filled(layers, pages, heads, page, D, dtype=torch.float16, seed=i) for i in range(2)], src, dst)
        check(ops, [filled(layers, pages, heads, page, D, dtype=torch.int8, seed=i) for i in range(2)] +
              [filled(layers, pages, heads, page // 16, dtype=torch.float32, seed=i) for i in range(2)], src, dst)


@pytest.mark.parametrize("n", [31, 32, 33, 480, 481, 1500])
def test_numbers_of_pairs(ops, n):
    """Around what one launch takes along; one page to many, too."""
    x = filled(2, 2 * n + 1, 3, 4)
    check(ops, [x], list(range(n)), list(range(n + 1, 2 * n + 1)))
    check(ops, [x], [2 * n] * n, list(range(n)))


@pytest.mark.parametrize("bytes_", [1, 3, 4, 12, 16, 100, 4095, 4096, 4097, 4100, 16384, 16400, 40003])
def test_page_sizes(ops, bytes_):
    """Any number of bytes, and pages that start anywhere."""
    check(ops, [filled(3, 10, bytes_, 1, seed=bytes_)], [0, 5, 9], [1, 2, 3])
    wide = filled(3, 10, bytes_ + 13, 1, seed=bytes_)
    before = wide.clone()
    view = wide[:, :, 7:7 + bytes_]
    check(ops, [view], [0, 5, 9], [1, 2, 3])
    before[:, [1, 2, 3], 7:7 + bytes_] = before[:, [0, 5, 9], 7:7 + bytes_]
    assert torch.equal(wide, before), "bytes beside the pages were written"


def test_interleaved_and_strided(ops):
    """Keys and values in one buffer, layers in another order, one layer of a cache, other integers."""
    both = filled(4, 30, 2, 8, 16, 64, dtype=torch.int16)
    before = both.clone()
    ops.paged_copy([both[:, :, 0], both[:, :, 1]], np.array([3, 4]), torch.tensor([7, 8]))
    before[:, [7, 8]] = before[:, [3, 4]]
    assert torch.equal(both, before)
    ops.paged_copy([both[2:3, :, 0]], (1,), (2,))
    before[2, 2, 0] = before[2, 1, 0]
    assert torch.equal(both, before)
    ops.paged_copy([both.transpose(0, 1).contiguous().transpose(0, 1)], [], [])
    check(ops, [both[1:].transpose(0, 1).contiguous().transpose(0, 1)[..., 0, :, :, :]], [5], [6])


def test_beyond_four_gigabytes(ops):
    x = torch.zeros(2, 1300, 1 << 21, dtype=torch.uint8, device="cuda")  # 5.5 GB
    x[1, 1299] = 7
    x[0, 1298] = 3
    ops.paged_copy([x], [1299, 1298], [0, 1])
    assert (x[1, 0] == 7).all() and (x[0, 1] == 3).all() and (x[0, 0] == 0).all() and (x[1, 1] == 0).all()


def test_capture_and_other_stream(ops):
    x = filled(2, 8, 4096, 1)
    first = x.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        ops.paged_copy([x], [0, 1], [4, 5])
    assert torch.equal(x, first)
    for _ in range(2):
        x[:, 0] += 1
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(x[:, 4:6], x[:, 0:2])
    with torch.cuda.stream(side):
        ops.paged_copy([x], [2], [3])
    side.synchronize()
    assert torch.equal(x[:, 2], x[:, 3])


def test_nothing_to_do(ops):
    x = filled(2, 8, 64, 1)
    before = x.clone()
    ops.paged_copy([x], [], [])
    ops.paged_copy([x], [3, 3], [3, 3])
    ops.paged_copy([x[:0]], [3], [4])
    torch.cuda.synchronize()
    assert torch.equal(x, before)


@pytest.mark.parametrize("src,dst", [([0], [8]), ([-1], [0]), ([8], [0]), ([0, 1], [2, 2]), ([0, 2], [2, 3]), ([0], [1, 2]),
                                     ([1 << 40], [0]), ([2, 0], [3, 2])])
def test_refused_pairs(ops, src, dst):
    x = filled(2, 8, 64, 1)
    before = x.clone()
    with pytest.raises(ValueError):
        ops.paged_copy([x], src, dst)
    torch.cuda.synchronize()
    assert torch.equal(x, before)


def test_refused_arrays(ops):
    x = filled(2, 8, 4, 64)
    for arrays in ([], [x[0, 0]], [x.cpu()], [x, x[:, :4]], [x.transpose(2, 3)], [x] * 9, [x[:, :1].expand(2, 8, 4, 64)],
                   [x[:1].expand(2, 8, 4, 64)]):
        with pytest.raises(ValueError):
            ops.paged_copy(arrays, [0], [1])
    with pytest.raises(TypeError):
        ops.paged_copy([x], [0.5], [1])
