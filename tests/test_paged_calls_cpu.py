"""What the paged operators' Python entries make of their arguments, as far as it shows without a GPU."""
import ctypes as C

import pytest
import torch

from trifuse_b200 import ops


def read_back(desc):
    """Page ids of a table's descriptor as the kernels would find them."""
    return [[C.c_int32.from_address(desc.ids + 4 * (r * desc.stride + c)).value for c in range(desc.columns)]
            for r in range(desc.requests)]


@pytest.mark.parametrize("make", ["plain", "rows apart", "one row", "expanded", "overlapping", "one expanded row",
                                  "every second row"])
def test_page_table_rows_are_found_where_they_are(make):
    base = torch.arange(100, 160, dtype=torch.int32)
    table = {"plain": base[:21].view(3, 7), "rows apart": base[:40].view(4, 10)[:, 2:7], "one row": base[None, 3:9],
             "expanded": base[None, :7].expand(5, 7), "overlapping": base.as_strided((4, 6), (2, 1)),
             "one expanded row": base[None, :7].expand(1, 7), "every second row": base.view(6, 10)[::2]}[make]
    desc = ops._page_table(table)
    assert desc.stride >= desc.columns and (desc.requests, desc.columns) == tuple(table.shape)
    held = getattr(desc, "tensor", table).untyped_storage()
    last = desc.ids + 4 * ((desc.requests - 1) * desc.stride + desc.columns)
    assert held.data_ptr() <= desc.ids and last <= held.data_ptr() + held.nbytes(), "read past the storage"
    assert read_back(desc) == table.tolist()


def test_a_plans_vectors_are_ordered_where_they_are_asked_for(monkeypatch):
    """positions and requests lie in the table that is still on its way: on another stream than the upload's they are
    ordered after it, as paged_attention orders itself."""
    plan = object.__new__(ops.PagedPlan)
    plan.made_on, plan.device_index = 7, 0
    plan._positions, plan._requests = torch.arange(3), torch.zeros(3)
    ordered = []
    monkeypatch.setattr(ops.PagedPlan, "order", lambda self, handle: ordered.append(handle))
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda device: 7, raising=False)
    assert plan.positions is plan._positions and plan.requests is plan._requests and not ordered
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda device: 8, raising=False)
    assert plan.positions is plan._positions and ordered == [8]
    assert plan.requests is plan._requests and ordered == [8, 8]


def test_no_plan_is_made_inside_a_capture(monkeypatch):
    """A captured upload would copy from a host buffer that other plans have since filled."""
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="captures a graph"):
        ops.PagedPlan([1], [4], 4, 2, 64, 16)


@pytest.mark.parametrize("scale", [2.4e38, 3.0e38, float("inf"), float("nan"), 0.0, -1.0, 1e-60])
def test_scales_that_overflow_inside_are_refused(scale):
    """The kernels fold log2(e) into the scale: beyond 2.3e38 every score would be 0 * inf."""
    from trifuse_b200._lib import PagedKV, PageTable, lib
    from tests.test_paged_cpu import plan
    _, d, _ = plan([1], [40])
    kv, tab = PagedKV(0x1000, 0x2000, 4, 2 * 16 * 128, 2, 16, 128, 1), PageTable(0x3000, 3, 1, 3)
    assert lib().tf_paged_attention(C.c_void_p(0x4000), 1024, C.byref(tab), C.byref(kv), C.byref(d), C.c_void_p(0x5000),
                                    scale, 1, C.c_void_p(0x6000), C.c_void_p(0x7000), 1 << 20, None) == 1


@pytest.fixture
def host_plans(monkeypatch):
    """Plans as far as the host makes them: the tables' allocations by size, none of them pinned."""
    sizes, empty = [], torch.empty

    def allocate(n, pin_memory=False, **kw):
        sizes.append(n)
        if n > 1 << 26:
            raise MemoryError(n)
        return empty(n, **kw)

    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch, "empty", allocate)
    return sizes


@pytest.mark.parametrize("new,kv,H,Hk", [([1 << 30], [1], 8, 2), ([1, -5], [1, 1], 8, 2), ([1], [1], 1 << 30, 1 << 30),
                                         ([(1 << 31) - 1] * 4, [1] * 4, 8, 2)])
def test_nothing_large_is_allocated_for_a_plan_that_is_refused(host_plans, new, kv, H, Hk):
    """The planner's refusal, not one of the allocator after gigabytes of pinned memory."""
    from trifuse_b200 import TriFuseError
    with pytest.raises((ValueError, TriFuseError)):
        ops.PagedPlan(new, kv, H, Hk, 128, 16)
    assert max(host_plans) <= 1 << 23


def test_a_plan_larger_than_the_first_allocation(host_plans):
    """800,000 rows: the table is made again at the size that the planner gives."""
    with pytest.raises((RuntimeError, AssertionError)):  # the upload, where there is no device
        ops.PagedPlan([400000, 400000], [400000, 500000], 8, 8, 128, 16, device="cuda:99")
    assert len(host_plans) == 2 and host_plans[0] <= 1 << 23 and host_plans[1] >= 8 * 800000


@pytest.mark.parametrize("lengths", [[2.5], [1.0], ["1"], [None]])
def test_lengths_that_are_no_integers_are_refused(host_plans, lengths):
    for new, kv in ((lengths, [40]), ([1], lengths)):
        with pytest.raises(TypeError):
            ops.PagedPlan(new, kv, 4, 2, 64, 16)


@pytest.mark.parametrize("make", ["one head, slots first", "one page of a wide buffer", "one page, expanded", "plain"])
def test_strides_of_single_heads_and_pages_do_not_matter(make):
    """A page that is contiguous is taken, whatever stride its dimensions of one carry."""
    base = torch.zeros(4, 16, 2, 64, dtype=torch.float16)
    k = {"one head, slots first": base[..., :1, :].contiguous().transpose(1, 2),
         "one page of a wide buffer": base.view(-1).as_strided((1, 2, 16, 64), (8, 1024, 64, 1)),
         "one page, expanded": base[0].reshape(2, 16, 64)[None].expand(1, 2, 16, 64),
         "plain": base.view(4, 2, 16, 64)}[make]
    d = ops._paged_kv(k, k)
    assert (d.pages, d.kv_heads, d.page_size, d.head_dim) == tuple(k.shape) and d.k == k.data_ptr()
    assert d.page_stride >= d.kv_heads * 16 * 64 and (d.pages == 1 or d.page_stride == k.stride(0))
    with pytest.raises(ValueError):
        ops._paged_kv(base.transpose(1, 2), base.transpose(1, 2))  # two heads inside each slot
