"""The page table of a paged key-value cache on the host: what it refuses, that a refused call changes
nothing, and what it marks for the device.  Built from the library's own header with the host compiler."""
import ctypes
import subprocess
from pathlib import Path

import numpy as np
import pytest

ROOT = Path(__file__).resolve().parent.parent
SZ, VP, U32P = ctypes.c_size_t, ctypes.c_void_p, ctypes.POINTER(ctypes.c_uint32)


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    so = tmp_path_factory.mktemp("paged") / "libpaged_host.so"
    subprocess.run(["g++", "-O1", "-std=c++17", "-fPIC", "-shared", str(ROOT / "tests" / "paged_host.cpp"), "-o", str(so)],
                   check=True)
    lib = ctypes.CDLL(str(so))
    for name, args in {"new": [SZ] * 4 + [ctypes.POINTER(VP)], "free": [VP], "assign": [VP, SZ, U32P, SZ],
                       "set_lens": [VP, U32P, SZ], "check_store": [VP, SZ, SZ, SZ],
                       "check_evict": [VP, VP, SZ, SZ, SZ], "shared": [VP], "words": [VP, U32P],
                       "changed": [VP, ctypes.POINTER(SZ)]}.items():
        getattr(lib, "pt_" + name).argtypes = args
    lib.pt_error.restype = ctypes.c_char_p
    lib.pt_shared.restype = SZ
    return lib


def words(a):
    a = np.ascontiguousarray(a, dtype=np.uint32)
    return a, a.ctypes.data_as(U32P)


class HostTable:
    def __init__(self, lib, seqs, per, page, pages):
        self.lib, self.size = lib, seqs * (per + 1)
        self.h = VP()
        self.call("new", seqs, per, page, pages, ctypes.byref(self.h))

    def call(self, name, *args):
        if getattr(self.lib, "pt_" + name)(*args):
            raise ValueError(self.lib.pt_error().decode())

    def assign(self, seq, ids):
        a, p = words(ids)
        self.call("assign", self.h, seq, p, a.size)

    def set_lens(self, lens):
        a, p = words(lens)
        self.call("set_lens", self.h, p, a.size)

    def store(self, first, count, m):
        self.call("check_store", self.h, first, count, m)

    def evict(self, to, keep, sinks=0, recent=0):
        self.call("check_evict", self.h, to.h, keep, sinks, recent)

    @property
    def shared(self):
        return self.lib.pt_shared(self.h)

    @property
    def words(self):
        a, p = words(np.zeros(self.size))
        self.lib.pt_words(self.h, p)
        return a

    def changed(self):
        out = (SZ * 3)()
        self.lib.pt_changed(self.h, out)
        return tuple(out)


@pytest.fixture
def table(host):
    made = []

    def make(*shape):
        made.append(HostTable(host, *shape))
        return made[-1]
    yield make
    for t in made:
        host.pt_free(t.h)


@pytest.mark.parametrize("shape", [(0, 1, 1, 1), (4097, 1, 1, 1), (1, 0, 1, 1), (1, 1, 0, 1), (1, 1, 1, 0),
                                   (1, 1 << 16, 1 << 15, 4), (1, 2, (1 << 64) - 1, 4), (2, (1 << 64) - 1, 1, 4),
                                   (1, 1, 1, 1 << 31), (4096, 1 << 20, 1, 4)])
def test_impossible_tables_are_refused(host, shape):
    with pytest.raises(ValueError):
        HostTable(host, *shape)


def test_bad_pages_are_refused_and_change_nothing(table):
    t = table(2, 3, 16, 10)
    t.assign(0, [9, 0, 4])
    t.set_lens([48, 0])
    before = t.words
    for seq, ids in [(2, [1]), (0, [1, 2, 3, 5]), (1, [10]), (1, [0xFFFFFFFF]), (1, [3, 3]), (0, [9, 0]), (0, [])]:
        with pytest.raises(ValueError):
            t.assign(seq, ids)
    for lens in ([49, 0], [48, 1], [48], [48, 0, 0], [0xFFFFFFFF, 0]):
        with pytest.raises(ValueError):
            t.set_lens(lens)
    np.testing.assert_array_equal(t.words, before)
    np.testing.assert_array_equal(before, [48, 0, 9, 0, 4, 0, 0, 0])


def test_only_changed_words_are_marked(table):
    t = table(3, 4, 8, 64)
    t.changed()
    t.assign(1, [5, 6])
    assert t.changed() == (3 + 4, 3 + 6, 1)
    t.assign(1, [5, 6, 7])  # a sequence that grew: its new page alone
    assert t.changed() == (3 + 6, 3 + 7, 1)
    t.set_lens([0, 17, 0])
    assert t.changed() == (1, 2, 1)
    t.set_lens([0, 17, 0])
    assert t.changed() == (0, 0, 0)
    t.assign(1, [5, 6, 7])
    assert t.changed() == (0, 0, 0)
    t.set_lens([0, 18, 0])  # a length and a page far behind it: two ranges, not all between
    t.assign(2, [9])
    assert t.changed() == (1, 3 + 9, 2)


def test_growing_a_sequence_checks_the_new_pages(table):
    t = table(2, 20, 4, 64)
    t.assign(0, [1, 2])
    t.assign(1, [3])
    for ids in ([1, 2, 2], [1, 2, 1], [1, 2, 5, 5], [1, 2, 64], [1, 2, 5, 6, 5]):
        with pytest.raises(ValueError):
            t.assign(0, ids)
    t.assign(0, [1, 2, 3])  # sequence 1's: shared now
    assert t.shared == 1
    t.assign(0, [1, 2, 3, 4])
    t.assign(0, [1, 2, 3, 4, *range(10, 26)])
    assert t.shared == 1
    t.assign(0, [1, 2])
    assert t.shared == 0
    t.assign(0, [2, 1])
    t.set_lens([8, 4])
    np.testing.assert_array_equal(t.words[2:4], [2, 1])


def test_many_small_changes_stay_few_ranges(table):
    t = table(4096, 1, 1, 4096)
    for i in range(4096):
        t.assign(i, [i])
    t.changed()
    for step in range(4):  # 2048 ranges of one word each time
        t.set_lens([i % 2 * ((step + 1) % 2) for i in range(4096)])
    first, last, ranges = t.changed()
    assert first <= 1 and last == 4096 and ranges <= 4096


def test_shared_pages_are_counted_through_reassignment(table):
    t = table(3, 3, 4, 8)
    t.assign(0, [1, 2])
    t.assign(1, [1, 3])
    assert t.shared == 1
    t.assign(2, [1, 3, 4])
    assert t.shared == 2
    t.assign(1, [5])
    assert t.shared == 1
    t.assign(2, [])
    assert t.shared == 0


def test_a_store_into_a_shared_page_is_refused(table):
    t = table(2, 3, 4, 8)
    t.assign(0, [1, 2, 3])
    t.assign(1, [1, 4])
    t.set_lens([9, 5])
    t.store(0, 2, 1)       # slots 8 and 4: pages 3 and 4
    t.store(0, 1, 5)       # slots 4..8
    with pytest.raises(ValueError):
        t.store(0, 1, 6)   # slot 3, in the shared page
    with pytest.raises(ValueError):
        t.store(1, 1, 99)  # all of sequence 1
    t.store(0, 2, 0)
    for first, count in [(3, 0), (2, 1), (0, 3), (1, (1 << 64) - 1)]:
        with pytest.raises(ValueError):
            t.store(first, count, 1)
    with pytest.raises(ValueError):
        t.store(0, 1, 1 << 31)


def test_evictions_that_cannot_be_done_are_refused(table):
    a, b = table(2, 4, 4, 16), table(2, 2, 4, 16)
    a.assign(0, [0, 1, 2, 3])
    a.assign(1, [4])
    a.set_lens([15, 2])
    b.assign(0, [8, 9])
    b.assign(1, [10])
    a.evict(b, 8, 4, 4)
    for keep, sinks, recent in [(0, 0, 0), (9, 0, 0), (8, 9, 0), (8, 4, 5), (8, 1, (1 << 64) - 1), (1 << 31, 0, 0)]:
        with pytest.raises(ValueError):
            a.evict(b, keep, sinks, recent)
    with pytest.raises(ValueError):
        a.evict(a, 8)
    for shape in [(1, 4, 4, 16), (2, 4, 8, 16), (2, 4, 4, 17)]:
        with pytest.raises(ValueError):
            a.evict(table(*shape), 1)
    b.assign(1, [9])       # page 9 is listed twice, and sequence 1 would be written to it
    for keep in (8, 4):
        with pytest.raises(ValueError):
            a.evict(b, keep)
    b.assign(1, [4])       # a page that tokens come from
    with pytest.raises(ValueError):
        a.evict(b, 8)
    b.assign(1, [11])
    a.evict(b, 8)
