"""A cache whose resizing runs out of memory half way: what is left is a cache, with the requests' tokens."""
import pytest
import torch

from trifuse_b200.paged import PagedCache


@pytest.mark.parametrize("dtype,arrays", [(torch.float16, 2), (torch.int8, 4)])
@pytest.mark.parametrize("pages", [7, 30])
@pytest.mark.parametrize("failing", [0, 1, 2, 3])
def test_memory_that_ends_half_way(monkeypatch, dtype, arrays, pages, failing):
    c = PagedCache(2, 12, 3, 16, 64, device="cpu", dtype=dtype)
    c.grow([0, 1], [40, 30])
    for t in c.arrays():
        t.view(torch.uint8).random_(generator=torch.Generator().manual_seed(1))
    held = {r: [t[:, c.pages[r]].clone() for t in c.arrays()] for r in (0, 1)}
    calls = []
    make = torch.Tensor.new_empty

    def new_empty(self, *a, **kw):
        calls.append(0)
        if len(calls) > failing:
            raise torch.OutOfMemoryError("no memory")
        return make(self, *a, **kw)

    monkeypatch.setattr(torch.Tensor, "new_empty", new_empty)
    if failing < arrays:
        with pytest.raises(torch.OutOfMemoryError):
            c.resize(pages)
    else:
        c.resize(pages)
    monkeypatch.undo()
    have = {t.shape[1] for t in c.arrays()}
    assert len(have) == 1
    have = have.pop()
    assert have == (pages if failing >= arrays else 12 if failing == 0 else min(pages, 12))
    used = [p for r in (0, 1) for p in c.pages[r]]
    assert sorted(used + c.free) == list(range(have))
    for r in (0, 1):
        assert all(torch.equal(a.view(torch.uint8), t[:, c.pages[r]].view(torch.uint8)) for a, t in zip(held[r], c.arrays()))
    c.grow([0], [16])
    c.resize(9)
    assert all(t.shape[1] == 9 for t in c.arrays()) and len(c.free) == 9 - 6
