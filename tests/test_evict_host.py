"""Which slots an eviction's search keeps, on the host: both forms of the search (a CTA alone, a cluster), with the
order and the counting rule of the library's own header, against the rule by sorting."""
import ctypes
import subprocess
from pathlib import Path

import numpy as np
import pytest

ROOT = Path(__file__).resolve().parent.parent
LARGEST = np.finfo(np.float32).max


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    so = tmp_path_factory.mktemp("evict") / "libevict_host.so"
    subprocess.run(["g++", "-O1", "-std=c++17", "-fPIC", "-shared", str(ROOT / "tests" / "evict_host.cpp"), "-o", str(so)],
                   check=True)
    lib = ctypes.CDLL(str(so))
    f32, u32 = (ctypes.POINTER(t) for t in (ctypes.c_float, ctypes.c_uint32))
    lib.ev_order.argtypes, lib.ev_order.restype = [ctypes.c_float], ctypes.c_uint32
    lib.ev_kept.argtypes = [ctypes.c_int, f32, *[ctypes.c_int] * 4, u32]
    return lib


def kept(lib, one, w, keep, sinks, recent):
    w, out = np.ascontiguousarray(w, dtype=np.float32), np.full(keep, 0xFFFFFFFF, dtype=np.uint32)
    n = lib.ev_kept(one, w.ctypes.data_as(lib.ev_kept.argtypes[1]), w.size, keep, sinks, recent,
                    out.ctypes.data_as(lib.ev_kept.argtypes[6]))
    assert n == keep
    return out


def rule(w, keep, sinks, recent):
    n = len(w)
    held = list(range(sinks)) + list(range(n - recent, n))
    order = sorted(range(sinks, n - recent), key=lambda s: (np.isnan(w[s]), 0.0 if np.isnan(w[s]) else -float(w[s]), s))
    return np.sort(held + order[: keep - len(held)])


@pytest.mark.parametrize("one", [0, 1])
@pytest.mark.parametrize("sinks,recent", [(0, 0), (2, 10), (0, 3), (4, 0), (12, 8)])
@pytest.mark.parametrize("large", [np.inf, LARGEST, 2.0 ** 127, np.nextafter(np.float32(2.0 ** 127), np.float32(0))])
@pytest.mark.parametrize("count", [0, 1, 7, 8, 9, 20, 21, 300])
def test_large_weights(lib, one, sinks, recent, large, count):
    """Fewer of them than free places, as many, and more."""
    rng = np.random.default_rng(5)
    w = rng.exponential(size=300).astype(np.float32)
    w[rng.permutation(300)[:count]] = large
    np.testing.assert_array_equal(kept(lib, one, w, 20, sinks, recent), rule(w, 20, sinks, recent))


@pytest.mark.parametrize("one", [0, 1])
@pytest.mark.parametrize("values", [
    [np.inf, LARGEST, 2.0 ** 127, 1.0], [np.inf, -np.inf, np.nan, 0.0, -0.0], [-1.0, -LARGEST, -np.inf],
    [1e-45, -1e-45, 0.0, 1e-38], [0.25], [np.nan], [np.inf], [-np.inf]])
def test_mixtures(lib, one, values):
    rng = np.random.default_rng(6)
    for n, keep, sinks, recent in [(2, 1, 0, 0), (2, 1, 1, 0), (2, 1, 0, 1), (97, 96, 3, 40), (600, 512, 1, 64),
                                   (513, 40, 0, 39), (700, 350, 175, 175)]:
        w = rng.choice(np.array(values, dtype=np.float32), n)
        np.testing.assert_array_equal(kept(lib, one, w, keep, sinks, recent), rule(w, keep, sinks, recent))


def test_order(lib):
    """Between no slot (0) and a held one (all bits set), NaN lowest, strictly with the value."""
    ascending = [-np.inf, -LARGEST, -1.0, -1e-45, 0.0, 1e-45, 1.0, 2.0 ** 127, LARGEST, np.inf]
    orders = [lib.ev_order(np.nan)] + [lib.ev_order(w) for w in ascending]
    assert orders == sorted(set(orders)) and orders[0] == 1 and orders[-1] < 0xFFFFFFFF
    assert lib.ev_order(-0.0) == lib.ev_order(0.0)
