"""What a page table sends to the device: the device's copy follows, and no decode step, however many sequences it
has, sends more than its own words or a copy of 512 KB, which the host does not wait for."""
import ctypes
import subprocess
from pathlib import Path

import numpy as np
import pytest

ROOT = Path(__file__).resolve().parent.parent
SZ, VP, U32P = ctypes.c_size_t, ctypes.c_void_p, ctypes.POINTER(ctypes.c_uint32)


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    so = tmp_path_factory.mktemp("update") / "libpaged_update.so"
    subprocess.run(["g++", "-O1", "-std=c++17", "-fPIC", "-shared", str(ROOT / "tests" / "paged_update_host.cpp"),
                    "-o", str(so)], check=True)
    lib = ctypes.CDLL(str(so))
    for name, args in {"new": [SZ] * 4, "free": [VP], "assign": [VP, SZ, U32P, SZ], "set_lens": [VP, U32P, SZ],
                       "send": [VP, ctypes.POINTER(SZ)]}.items():
        getattr(lib, "pu_" + name).argtypes = args
    lib.pu_new.restype, lib.pu_free.restype = VP, None
    return lib


class Both:
    def __init__(self, lib, *shape):
        self.lib, self.h = lib, lib.pu_new(*shape)

    def __del__(self):
        self.lib.pu_free(self.h)

    def assign(self, seq, ids):
        a = np.ascontiguousarray(ids, dtype=np.uint32)
        self.lib.pu_assign(self.h, seq, a.ctypes.data_as(U32P), a.size)

    def set_lens(self, lens):
        a = np.ascontiguousarray(lens, dtype=np.uint32)
        self.lib.pu_set_lens(self.h, a.ctypes.data_as(U32P), a.size)

    def send(self):
        """(single words, words of a range); the device's copy is the table's."""
        out = (SZ * 2)()
        assert self.lib.pu_send(self.h, out)
        return tuple(out)


@pytest.mark.parametrize("seqs", [1, 64, 1900, 1921, 2500, 4096])
@pytest.mark.parametrize("together", [False, True])
def test_a_decode_step_sends_its_own_words(host, seqs, together):
    """Every sequence a token longer, with a new page where it needs one: sequences that began together (all need
    one in the same step), and apart."""
    page, per = 4, 64
    t = Both(host, seqs, per, page, seqs * per)
    lens = np.full(seqs, 5) if together else 1 + np.arange(seqs) * 7 % 100
    pages = [list(range(i * per, i * per - (-n // page))) for i, n in enumerate(lens.tolist())]
    for i in range(seqs):
        t.assign(i, pages[i])
    t.set_lens(lens)
    t.send()
    for _ in range(9):
        lens = lens + 1
        new = 0
        for i in range(seqs):
            if lens[i] > len(pages[i]) * page:
                pages[i].append(i * per + len(pages[i]))
                t.assign(i, pages[i])
                new += 1
        t.set_lens(lens)
        words, copied = t.send()
        assert (words == seqs + new and copied == 0) or (words == 0 and copied <= 1 << 17), (words, copied, new)


def test_the_device_follows_any_changes(host):
    rng = np.random.default_rng(3)
    seqs, per, page = 300, 100, 2
    t = Both(host, seqs, per, page, 500)
    assert t.send() == (0, 0)
    for step in range(60):
        t.set_lens(np.zeros(seqs))
        held = np.zeros(seqs, dtype=int)
        for i in rng.permutation(seqs)[: 1 + step * 5]:
            held[i] = rng.integers(0, per + 1)
            t.assign(i, rng.permutation(500)[: held[i]])
        t.set_lens(np.minimum(rng.integers(0, 2 * per, seqs), held * page))
        if step % 3:
            t.send()
    t.send()
    assert t.send() == (0, 0)


def test_what_was_set_back_is_not_sent(host):
    t = Both(host, 4096, 1, 1, 4096)
    for i in range(4096):
        t.assign(i, [i])
    t.send()
    for _ in range(5):
        t.set_lens(np.arange(4096) % 2)
        t.set_lens(np.zeros(4096))
    assert t.send() == (0, 0)
