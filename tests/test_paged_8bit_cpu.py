"""The operators of the 8-bit cache, page copies and beam selection as far as they show without a GPU: what is refused
before any launch, the descriptors of scales, the plans' list of requests whose codes are widened."""
import ctypes as C
import random
import struct

import pytest
import torch

from tests.test_paged_cpu import plan
from trifuse_b200 import ops
from trifuse_b200._lib import CopyArray, PagedKV, PagedPlanDesc, PagedScales, PageTable, lib

I8, E4M3 = 4, 5


def kv(pages=4, stride=None, heads=2, page=16, D=128, dtype=I8, k=0x1000, v=0x2000):
    return PagedKV(k, v, pages, heads * page * D if stride is None else stride, heads, page, D, dtype)


def scales(k=0x8000, v=0x9000, stride=2):
    return PagedScales(k, v, stride)


def append(kv_=None, sc=None, tab=None, rows=1, heads=8, act=1, qkv=0x4000, stride=12 * 128, qn=0, kn=0, eps=1e-5,
           theta=0.0, pos=0x6000, req=0x6100, out=0x7000):
    kv_, sc, tab = kv_ or kv(), sc or scales(), tab or PageTable(0x3000, 3, 1, 3)
    return lib().tf_paged_append_8bit(C.c_void_p(qkv), stride, rows, heads, act, C.c_void_p(qn), C.c_void_p(kn), eps,
                                      theta, C.c_void_p(pos), C.c_void_p(req), C.byref(tab), C.byref(kv_), C.byref(sc),
                                      C.c_void_p(out), None)


def attend(kv_=None, sc=None, tab=None, d=None, stride=1024, q=0x4000, ws=1 << 20, act=1, scale=0.1, out=0x6000):
    d = d or plan([1], [40])[1]
    kv_, sc, tab = kv_ or kv(), sc or scales(), tab or PageTable(0x3000, 3, 1, 3)
    return lib().tf_paged_attention_8bit(C.c_void_p(q), stride, C.byref(tab), C.byref(kv_), C.byref(sc), C.byref(d),
                                         C.c_void_p(0x5000), scale, act, C.c_void_p(out), C.c_void_p(0x7000), ws, None)


@pytest.mark.parametrize("call", [append, attend])
def test_caches_that_are_refused(call):
    assert call(kv_=kv(dtype=1)) == 8 and call(kv_=kv(dtype=3)) == 8      # not codes
    assert call(kv_=kv(page=8)) == 8                                      # below a block of tokens
    assert call(kv_=kv(D=96)) == 8 and call(kv_=kv(page=24)) == 8
    assert call(kv_=kv(stride=2 * 16 * 128 + 8)) == 2                     # codes are read 16 bytes at a time
    assert call(kv_=kv(stride=2 * 16 * 128 - 16)) == 2 and call(kv_=kv(pages=0)) == 2
    assert call(kv_=kv(k=0)) == 1 and call(kv_=kv(v=0x2008)) == 1
    assert call(sc=scales(k=0)) == 1 and call(sc=scales(v=0x9002)) == 1
    assert call(sc=scales(stride=1)) == 2 and call(sc=scales(stride=1 << 38)) == 2
    assert call(act=3) == 1 and call(act=4) == 1
    L = lib()
    tab = PageTable(0x3000, 3, 1, 3)
    none = C.POINTER(PagedScales)()
    d = plan([1], [40])[1]
    assert L.tf_paged_attention_8bit(0x4000, 1024, C.byref(tab), C.byref(kv()), none, C.byref(d), 0x5000, 0.1, 1, 0x6000,
                                     0x7000, 1 << 20, None) == 1
    assert L.tf_paged_append_8bit(0x4000, 1536, 1, 8, 1, 0, 0, 1e-5, 0.0, 0x6000, 0x6100, C.byref(tab), C.byref(kv()),
                                  none, 0x7000, None) == 1


def test_append_arguments():
    assert append(rows=-1) == 2 and append(stride=12 * 128 - 8) == 2 and append(stride=12 * 128 + 4) == 2
    assert append(heads=7) == 2 and append(qn=0x100) == 1 and append(qn=0x100, kn=0x200, eps=0.0) == 1
    assert append(theta=0.5) == 1 and append(qkv=0) == 1 and append(out=0x7008) == 1 and append(pos=0) == 1
    assert append(tab=PageTable(0x3000, 2, 1, 3)) == 2
    assert append(rows=0) == 0


def test_attention_arguments():
    assert attend(q=0) == 1 and attend(out=0x6010) == 1 and attend(stride=1000) == 2 and attend(scale=0.0) == 1
    assert attend(tab=PageTable(0x3000, 2, 1, 2)) == 2 and attend(kv_=kv(page=32)) == 2
    many = plan([300], [300])[1]
    tab = PageTable(0x3000, 19, 1, 19)
    assert many.widened_bytes > 0
    assert attend(d=many, tab=tab, ws=many.workspace_bytes + many.widened_bytes - 1) == 1


def widened(d, table):
    first = struct.unpack_from(f"{d.requests}i", table, d.widened_offset)
    at = d.widened_offset + -(-4 * d.requests // 16) * 16
    return first, [struct.unpack_from("4i", table, at + 16 * i)[:3] for i in range(d.widened_requests)]


@pytest.mark.parametrize("seed", range(6))
def test_the_list_of_widened_requests(seed):
    """Requests with more than 128 packed rows and a history, each page of theirs once, one after the other; the scratch
    holds their codes at two bytes and their scales."""
    rng = random.Random(seed)
    H, Hk = rng.choice([(8, 2), (4, 4), (16, 1)])
    D, page = rng.choice([64, 128]), rng.choice([16, 64, 256])
    new = [rng.choice([0, 1, 7, 40, 128, 129, 600]) for _ in range(rng.randint(1, 20))]
    kv_ = [rng.choice([0, 1, n, n + 1, n + 5000]) for n in new]
    _, d, table = plan(new, kv_, H, Hk, D, page)
    want = [r for r, (n, L) in enumerate(zip(new, kv_)) if n * H // Hk > 128 and L > 0]
    assert d.widened_requests == len(want)
    if not any(n * H // Hk > 128 for n in new):
        assert d.widened_bytes == d.widened_pages == 0
        return
    first, requests = widened(d, table)
    at = 0
    for r, (p, request, length) in zip(want, requests):
        assert (p, request, length) == (at, r, kv_[r]) and first[r] == at
        at += -(-kv_[r] // page)
    assert d.widened_pages == at and all(first[r] == -1 for r in range(len(new)) if r not in want)
    if at:
        assert d.widened_bytes >= 2 * at * Hk * page * D * 2 + 2 * at * Hk * page // 16 * 4


def test_pages_below_a_block_are_not_widened():
    d = plan([300], [300], page=8)[1]
    assert d.widened_bytes == d.widened_requests == 0


@pytest.mark.parametrize("make", ["plain", "pages apart", "one page, expanded", "one head, blocks first", "one block"])
def test_strides_of_scales(make):
    base = torch.zeros(4, 3, 6)
    s = {"plain": base, "pages apart": torch.zeros(4, 2, 3, 6)[:, 0], "one page, expanded": base[:1].expand(1, 3, 6),
         "one head, blocks first": torch.zeros(4, 6, 1).transpose(1, 2), "one block": torch.zeros(4, 3, 1)}[make]
    cache = PagedKV(0x1000, 0x2000, s.shape[0], 1 << 20, s.shape[1], s.shape[2] * 16, 64, I8)
    d = ops._paged_scales(s, s, cache)
    assert d.k == s.data_ptr() and (s.shape[0] == 1 or d.page_stride == s.stride(0))
    assert d.page_stride >= s.shape[1] * s.shape[2]


def test_scales_that_are_refused():
    cache = PagedKV(0x1000, 0x2000, 4, 1 << 20, 3, 96, 64, I8)
    good = torch.zeros(4, 3, 6)
    for k, v in ((good, None), (None, good), (good.double(), good), (good, good[:3]), (good[..., :5], good[..., :5]),
                 (torch.zeros(4, 6, 3).transpose(1, 2), good), (torch.zeros(4, 2, 3, 6)[:, 0], good),
                 (torch.zeros(4, 3, 12)[..., ::2],) * 2, (torch.zeros(3, 4, 6).transpose(0, 1),) * 2):
        with pytest.raises(ValueError):
            ops._paged_scales(k, v, cache)
    codes = torch.zeros(4, 3, 96, 64, dtype=torch.int8)
    with pytest.raises(ValueError, match="k_scales"):
        ops._paged_kv(codes, codes)
    with pytest.raises(ValueError, match="int8 or float8"):
        ops._paged_kv(codes.half(), codes.half(), ops._CODES)


def copy(arrays, src, dst, layers=2, pages=8, count=None):
    a = (CopyArray * max(len(arrays), 1))(*arrays)
    n = len(src)
    return lib().tf_paged_copy(a, len(arrays) if count is None else count, layers, pages, (C.c_int32 * max(n, 1))(*src),
                               (C.c_int32 * max(n, 1))(*dst), n, None)


def test_copies_that_are_refused():
    good = CopyArray(0x1000, 8 * 64, 64, 64)
    for src, dst in (([0], [8]), ([-1], [0]), ([0, 1], [2, 2]), ([0, 2], [2, 3]), ([2, 0], [3, 2]), ([1, 1, 3], [2, 4, 1])):
        assert copy([good], src, dst) == 1
    assert copy([CopyArray(0, 8 * 64, 64, 64)], [0], [1]) == 1
    assert copy([CopyArray(0x1000, 8 * 64, 32, 64)], [0], [1]) == 2
    assert copy([CopyArray(0x1000, -64, 64, 64)], [0], [1]) == 2 and copy([CopyArray(0x1000, 64, 64, -1)], [0], [1]) == 2
    assert copy([good] * 9, [0], [1]) == 1 and copy([good], [0], [1], count=-1) == 1
    assert copy([good], [0], [1], layers=-1) == 2 and copy([good], [0], [1], pages=1 << 31) == 2
    # Nothing to do: no launch.
    assert copy([good], [], []) == 0 and copy([good], [3, 3, 0], [3, 3, 0]) == 0
    assert copy([good], [0], [1], layers=0) == 0 and copy([], [0], [1]) == 0


def test_beams_that_are_refused():
    L = lib()
    size = C.c_size_t()
    for args, error in (((1, 4, 100, 4), 0), ((-1, 4, 100, 4), 2), ((1, 0, 100, 4), 2), ((1, 65, 100, 4), 2),
                        ((1, 4, 0, 4), 2), ((1, 4, 100, 0), 1), ((1, 4, 100, 65), 1), (((1 << 24) + 1, 4, 100, 4), 2)):
        assert L.tf_beam_select_workspace_size(*args, C.byref(size)) == error
    assert L.tf_beam_select_workspace_size(1, 4, 100, 4, None) == 1

    def select(logits=0x1000, stride=100, R=2, beams=4, V=100, dtype=3, scores=0x2000, count=4, score=0x3000,
               parent=0x4000, token=0x5000, ws=0x6000, nbytes=1 << 20):
        return L.tf_beam_select(logits, stride, R, beams, V, dtype, scores, None, -1, count, score, parent, token, ws, nbytes,
                                None)

    assert select(dtype=4) == 1 and select(stride=99) == 2 and select(logits=0) == 1 and select(logits=0x1002) == 1
    assert select(scores=0) == 1 and select(score=0) == 1 and select(parent=0) == 1 and select(token=0) == 1
    assert select(ws=0) == 1 and select(ws=0x6008) == 1 and select(nbytes=8) == 1
    assert select(R=0) == 0
    for R, beams, V, count in ((2, 4, 100, 4), (3, 64, 7, 64)):
        assert L.tf_beam_select_workspace_size(R, beams, V, count, C.byref(size)) == 0
        assert size.value == R * beams * (16 + 8 * min(count, V))  # as the Python entry allocates
