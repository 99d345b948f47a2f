"""The planner of paged attention, on the host: every query row meets every key tile exactly once, whatever the
lengths, and what cannot be planned is refused before anything runs."""
import ctypes as C
import random

import pytest

from trifuse_b200._lib import PagedKV, PagedPlanDesc, PageTable, lib


def plan(new, kv, H=8, Hk=2, D=128, page=16):
    n = len(new)
    a, b = (C.c_int32 * n)(*new), (C.c_int32 * n)(*kv)
    d = PagedPlanDesc()
    status = lib().tf_paged_plan_make(a, b, n, H, Hk, D, page, C.byref(d), None, 0)
    if status != 10:  # the size is known, the table was not given
        return status, None, None
    table = (C.c_uint8 * d.table_bytes)()
    assert lib().tf_paged_plan_make(a, b, n, H, Hk, D, page, C.byref(d), table, d.table_bytes) == 0
    return 0, d, bytes(table)


@pytest.mark.parametrize("new,kv,error", [([-1], [4], 2), ([1], [-4], 2), ([1 << 30], [1], 8), ([1], [(1 << 30) + 1], 8)])
def test_lengths_refused(new, kv, error):
    assert plan(new, kv)[0] == error


@pytest.mark.parametrize("geometry,error", [(dict(H=7, Hk=2), 2), (dict(H=0), 2), (dict(D=96), 8), (dict(page=24), 8),
                                            (dict(page=4), 8), (dict(page=512), 8), (dict(H=256, Hk=2), 8)])
def test_geometry_refused(geometry, error):
    assert plan([1], [4], **geometry)[0] == error


def test_table_capacity():
    _, d, _ = plan([1, 2], [5, 600])
    a, b = (C.c_int32 * 2)(1, 2), (C.c_int32 * 2)(5, 600)
    table = (C.c_uint8 * d.table_bytes)(*([7] * d.table_bytes))
    again = PagedPlanDesc()
    assert lib().tf_paged_plan_make(a, b, 2, 8, 2, 128, 16, C.byref(again), table, d.table_bytes - 1) == 10
    assert again.table_bytes == d.table_bytes and set(bytes(table)) == {7}
    assert lib().tf_paged_plan_make(a, b, 2, 8, 2, 128, 16, None, table, d.table_bytes) == 1
    assert lib().tf_paged_plan_make(a, b, 2, 8, 2, 128, 16, C.byref(again), None, 8) == 1
    assert lib().tf_paged_plan_make(None, b, 2, 8, 2, 128, 16, C.byref(again), None, 0) == 1


def test_attention_and_append_refuse_before_any_launch():
    L = lib()
    _, d, _ = plan([1], [40])
    kv = PagedKV(0x1000, 0x2000, 4, 2 * 16 * 128, 2, 16, 128, 1)
    tab = PageTable(0x3000, 3, 1, 3)

    def attend(kv=kv, tab=tab, stride=1024, q=0x4000, ws=1 << 20, act=1, scale=0.1, out=0x6000):
        return L.tf_paged_attention(C.c_void_p(q), stride, C.byref(tab), C.byref(kv), C.byref(d), C.c_void_p(0x5000),
                                    scale, act, C.c_void_p(out), C.c_void_p(0x7000), ws, None)

    assert attend(q=0) == 1 and attend(q=0x4008) == 1 and attend(out=0x6010) == 1
    assert attend(stride=1000) == 2 and attend(stride=1028) == 2
    assert attend(act=3) == 1 and attend(scale=-1.0) == 1
    assert attend(tab=PageTable(0x3000, 2, 1, 2)) == 2          # the request needs three pages
    assert attend(tab=PageTable(0x3000, 1, 1, 3)) == 2          # rows overlap
    assert attend(kv=PagedKV(0x1000, 0x2000, 4, 2 * 16 * 128, 2, 16, 128, 2)) == 8   # bf16 cache under f16
    assert attend(kv=PagedKV(0x1000, 0x2000, 4, 64, 2, 16, 128, 1)) == 2             # pages overlap
    assert attend(kv=PagedKV(0x1000, 0x2008, 4, 2 * 16 * 128, 2, 16, 128, 1)) == 1
    if d.workspace_bytes:
        assert attend(ws=d.workspace_bytes - 1) == 1

    def append(stride=12 * 128, rows=1, qn=None, kn=None, theta=1e4, pos=0x100):
        return L.tf_paged_append(C.c_void_p(0x4000), stride, rows, 8, 1, qn, kn, 1e-5, theta, C.c_void_p(pos),
                                 C.c_void_p(0x200), C.byref(tab), C.byref(kv), C.c_void_p(0x8000), None)

    assert append(stride=11 * 128) == 2 and append(rows=-1) == 2
    assert append(qn=C.c_void_p(0x100)) == 1 and append(theta=0.5) == 1 and append(pos=0) == 1
    assert append(rows=0) == 0


def segments(d, raw, kind):
    import struct
    blocks, first, at = (getattr(d, kind + name) for name in ("_blocks", "_starts_offset", "_segments_offset"))
    starts = struct.unpack_from(f"<{blocks + 1}i", raw, first)
    return [(b, struct.unpack_from("<13i", raw, at + 64 * i))
            for b in range(blocks) for i in range(starts[b], starts[b + 1])]


def test_every_row_meets_every_tile_once():
    rng = random.Random(5)
    for case in range(60):
        B = rng.randint(1, 40)
        new = [rng.choice([0, 1, 1, rng.randint(1, 400)]) for _ in range(B)]
        kv = [rng.choice([0, n, n + rng.randint(0, 20000), max(0, n - 3)]) for n in new]
        H, Hk = rng.choice([(16, 16), (8, 1), (14, 2), (32, 8)])
        _, d, raw = plan(new, kv, H, Hk)
        rows_seen = {}
        for kind, most, keys, all_parts in (("split", 16, 32, d.split_parts), ("half", 128, 128, d.half_parts),
                                            ("tile", 256, 128, d.tile_parts)):
            seen, parts, cut = {}, {}, set()
            load = {}
            for block, g in segments(d, raw, kind):
                q_row, n, L, req, head, row0, rows, t0, t1, part, part0, count, counter = g
                assert n == new[req] and L == kv[req] and q_row == sum(new[:req])
                assert 0 < rows <= most and row0 + rows <= n * (H // Hk)
                load[block] = load.get(block, 0) + t1 - t0
                seen.setdefault((req, head, row0, rows), []).append((t0, t1))
                if count > 1:
                    assert part0 <= part < part0 + count <= all_parts and part not in parts
                    parts[part] = counter
                    cut.add(part0)
                else:
                    assert part == -1
            assert len(parts) == all_parts
            assert len(cut) == (d.split_counters if kind == "split" else getattr(d, kind + "_merges"))
            assert len(load) <= (296 if kind == "half" else 148)
            for (req, head, row0, rows), spans in seen.items():
                spans.sort()
                last = kv[req] - new[req] + (row0 + rows - 1) // (H // Hk)
                assert spans[0][0] == 0 and spans[-1][1] == (0 if last < 0 else last // keys + 1)
                assert all(a[1] == b[0] for a, b in zip(spans, spans[1:]))
                rows_seen[(req, head)] = rows_seen.get((req, head), 0) + rows
        for r in range(B):
            for h in range(Hk):
                assert rows_seen.get((r, h), 0) == new[r] * (H // Hk)
