"""Paged key-value caches on the GPU against the formulas in 64 bits: store, single-token attention (with and
without its weights), eviction, and a run of them together as a decode loop makes it."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24  # half a step of f32


@pytest.fixture(scope="module")
def ops(slm, ctx):
    return slm.Ops(ctx)


def to_bf16(x):
    """Nearest bf16, ties to even, as 16-bit words (finite x)."""
    b = np.ascontiguousarray(x, dtype=np.float32).view(np.uint32)
    return ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)


def from_bf16(w):
    return (w.astype(np.uint32) << 16).view(np.float32)


class Pool:
    """Host pool [pages][key_heads][page][dh] and weights, its device buffers, and a table over them."""

    def __init__(self, slm, ctx, ops, rng, lens, key_heads, dh, page, bf16, spare=3, bad=None):
        self.slm, self.ctx, self.ops, self.bf16 = slm, ctx, ops, bf16
        self.kh, self.dh, self.page, self.lens = key_heads, dh, page, list(lens)
        per = [-(-n // page) for n in lens]
        self.per = max(1, max(per))
        self.pages = sum(per) + spare
        order = rng.permutation(self.pages)
        cuts = np.cumsum([0] + per)
        self.ids = [order[a:b].tolist() for a, b in zip(cuts[:-1], cuts[1:])]
        self.free = order[cuts[-1]:].tolist()
        shape = (self.pages, key_heads, page, dh)
        self.k, self.v = (rng.standard_normal(shape).astype(np.float32) for _ in range(2))
        self.w = rng.exponential(size=shape[:3]).astype(np.float32)
        if bf16:
            self.k, self.v = from_bf16(to_bf16(self.k)), from_bf16(to_bf16(self.v))
        if bad is not None:  # every row that no sequence holds
            held = np.zeros((self.pages, page), dtype=bool)
            for ids, n in zip(self.ids, lens):
                for s in range(n):
                    held[ids[s // page], s % page] = True
            for x in (self.k, self.v, self.w):
                x[~held.reshape(self.pages, 1, page).repeat(key_heads, 1)] = bad
        self.kb, self.vb = self.up(self.k), self.up(self.v)
        self.wb = ops.upload(self.w)
        self.table = slm.Table(ctx, len(self.lens), self.per, page, self.pages)
        for i, row in enumerate(self.ids):
            self.table.assign(i, row)
        self.table.set_lens(self.lens)

    def up(self, x):
        if not self.bf16:
            return self.ops.upload(x)
        b = np.ascontiguousarray(x, dtype=np.float32).view(np.uint32)
        return self.ops.upload((b >> 16).astype(np.uint16).reshape(-1).view(np.float32))

    def down(self, buf):
        x = buf.read()
        x = from_bf16(x.view(np.uint16)) if self.bf16 else x
        return x[: self.k.size].reshape(self.k.shape)

    def weights(self):
        return self.wb.read().reshape(self.w.shape)

    def rows(self, x, i, lo, hi):
        """Slots lo..hi-1 of sequence i: [key_heads][slots](dh)."""
        s = np.arange(lo, hi)
        return np.moveaxis(x[np.asarray(self.ids[i], dtype=int)[s // self.page], :, s % self.page], 0, 1)

    def attend(self, q, heads, scale, reach=None, weights=False, y=None, **more):
        y = y or self.ops.zeros(1)
        scores = self.ops.zeros(1)
        self.ops.paged_attend(y, scores, q, self.kb, self.vb, self.table, heads=heads, key_heads=self.kh, dh=self.dh,
                              scale=scale, reach=reach, bf16=self.bf16, weights=self.wb if weights else None, **more)
        n = len(self.lens) * heads * self.dh
        return y.read(n).reshape(len(self.lens), heads, self.dh)

    def formula(self, q, heads, scale, reach=None):
        """y, its tolerance, and per sequence (first visible slot, weights drawn, their tolerance)."""
        group = heads // self.kh
        y, tol, drawn = np.zeros((len(self.lens), heads, self.dh)), np.zeros((len(self.lens), heads, self.dh)), []
        for i, n in enumerate(self.lens):
            lo = max(0, n - reach) if reach else 0
            if n == 0:
                drawn.append((0, None, None))
                continue
            k, v = (self.rows(x, i, lo, n).astype(np.float64) for x in (self.k, self.v))
            qi = q[i].astype(np.float64).reshape(self.kh, group, self.dh)
            x = scale * np.einsum("hgd,hsd->hgs", qi, k)
            p = np.exp(x - x.max(-1, keepdims=True))
            p /= p.sum(-1, keepdims=True)
            y[i] = np.einsum("hgs,hsd->hgd", p, v).reshape(heads, self.dh)
            # A score is a sum of dh products of operands good to 2^-21 each, rounded dh times (four
            # standard deviations of independent roundings); its error enters p once directly and once
            # through the sum; sums over n tokens round n times.
            size = abs(scale) * np.einsum("hgd,hsd->hgs", abs(qi), abs(k)).max(-1)
            e = 2 * size * (2.0 ** -20 + (4 * np.sqrt(self.dh) + 4) * U) + (4 * np.sqrt(n - lo) + 16) * U + 2.0 ** -20
            tol[i] = (e[..., None] * np.einsum("hgs,hsd->hgd", p, abs(v))).reshape(heads, self.dh)
            drawn.append((lo, p.sum(1), (e[..., None] * p).sum(1)))
        return y, tol + 1e-30, drawn

    def check_weights(self, before, after, drawn, times=1):
        want, tol = before.astype(np.float64), np.zeros(before.shape)
        for i, (lo, add, err) in enumerate(drawn):
            if add is None:
                continue
            s = np.arange(lo, self.lens[i])
            at = (np.asarray(self.ids[i])[s // self.page], slice(None), s % self.page)
            want[at] += times * add.T
            tol[at] += times * err.T + times * 2 * U * abs(want[at])
        np.testing.assert_array_equal(after[tol == 0], before[tol == 0])
        assert (abs(after - want) <= tol).all()


# lens, heads, key_heads, dh, page, bf16, reach
ATTEND = [
    ([1], 1, 1, 8, 1, False, None),
    ([0, 1, 2, 15, 16, 17], 4, 2, 16, 16, False, None),
    ([33, 0, 0, 5], 6, 2, 24, 7, False, None),
    ([97], 12, 4, 64, 16, False, None),
    ([700, 31, 0, 1025], 12, 4, 64, 64, False, None),
    ([700, 31, 0, 1025], 12, 4, 64, 64, True, None),
    ([513, 512, 511, 1], 32, 8, 128, 32, True, None),
    ([513, 512, 511, 1], 32, 8, 128, 32, False, None),
    ([260, 19], 5, 5, 40, 24, True, None),
    ([260, 19], 9, 3, 80, 8, False, None),
    ([300, 1, 64], 16, 1, 256, 16, False, None),
    ([300, 1, 64], 17, 1, 256, 128, True, None),
    ([130, 129, 3], 24, 2, 96, 5, True, None),
    ([130, 129, 3], 20, 2, 136, 13, False, None),
    ([90, 1500], 7, 1, 192, 100, True, None),
    ([90, 700], 8, 1, 200, 3, False, None),
    ([40, 900, 0, 100], 12, 4, 64, 16, False, 100),
    ([40, 900, 0, 100], 16, 2, 128, 16, True, 1),
    ([4500], 12, 4, 64, 16, False, 4096),
    ([6000, 100], 6, 2, 32, 16, False, None),
    ([9, 0, 3000, 77, 1, 2, 500, 499, 64], 8, 8, 64, 64, True, None),
    ([30000] + [1] * 70, 1, 1, 64, 64, False, None),  # one sequence in pieces of nearly all warps
    ([30000] + [1] * 70, 2, 1, 64, 64, True, None),
    ([1 + i % 3 for i in range(700)], 3, 1, 16, 4, False, None),  # more pairs than warps
    ([(37 * i) % 400 for i in range(300)], 16, 8, 128, 16, True, None),
    ([(61 * i) % 700 for i in range(200)], 20, 4, 64, 16, False, 333),
]


@pytest.mark.parametrize("case", range(len(ATTEND)))
@pytest.mark.parametrize("weights", [False, True])
def test_attend(slm, ctx, ops, case, weights):
    lens, heads, kh, dh, page, bf16, reach = ATTEND[case]
    rng = np.random.default_rng(100 + case)
    pool = Pool(slm, ctx, ops, rng, lens, kh, dh, page, bf16)
    q = rng.standard_normal((len(lens), heads, dh)).astype(np.float32)
    scale = dh ** -0.5
    y, tol, drawn = pool.formula(q, heads, scale, reach)
    got = pool.attend(ops.upload(q), heads, scale, reach, weights)
    assert (abs(got - y) <= tol).all(), float((abs(got - y) / tol).max())
    if weights:
        pool.check_weights(pool.w, pool.weights(), drawn)
        again = pool.attend(ops.upload(q), heads, scale, reach, True)
        np.testing.assert_array_equal(again, got)
        pool.check_weights(pool.w, pool.weights(), drawn, times=2)


@pytest.mark.parametrize("bf16", [False, True])
def test_attend_at_every_head_size(slm, ctx, ops, bf16):
    for dh in range(8, 257, 8):
        rng = np.random.default_rng(dh)
        group, lens = 1 + dh // 8 % 18, [dh % 37 + 1, 0, 400 + dh]
        pool = Pool(slm, ctx, ops, rng, lens, 2, dh, 1 + dh % 29, bf16)
        q = rng.standard_normal((3, 2 * group, dh)).astype(np.float32)
        y, tol, drawn = pool.formula(q, 2 * group, dh ** -0.5)
        got = pool.attend(ops.upload(q), 2 * group, dh ** -0.5, weights=True)
        assert (abs(got - y) <= tol).all(), dh
        pool.check_weights(pool.w, pool.weights(), drawn)


@pytest.mark.parametrize("lens,page", [([1200003], 512), ([i % 5 for i in range(4096)], 2)])
def test_attend_at_the_ends_of_the_range(slm, ctx, ops, lens, page):
    rng = np.random.default_rng(17)
    pool = Pool(slm, ctx, ops, rng, lens, 1, 8, page, True)
    q = rng.standard_normal((len(lens), 2, 8)).astype(np.float32)
    y, tol, drawn = pool.formula(q, 2, 0.35)
    got = pool.attend(ops.upload(q), 2, 0.35, weights=True)
    assert (abs(got - y) <= tol).all(), float((abs(got - y) / tol).max())
    pool.check_weights(pool.w, pool.weights(), drawn)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("scale", [3.0, -0.5, 0.0])
def test_attend_with_peaked_and_flat_scores(slm, ctx, ops, bf16, scale):
    rng = np.random.default_rng(7)
    pool = Pool(slm, ctx, ops, rng, [600, 37], 2, 64, 16, bf16)
    q = rng.standard_normal((2, 6, 64)).astype(np.float32)
    y, tol, drawn = pool.formula(q, 6, scale)
    got = pool.attend(ops.upload(q), 6, scale, weights=True)
    assert (abs(got - y) <= tol).all(), float((abs(got - y) / tol).max())
    pool.check_weights(pool.w, pool.weights(), drawn)


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf, np.finfo(np.float32).max])
@pytest.mark.parametrize("bf16", [False, True])
def test_rows_outside_the_sequences_are_not_read(slm, ctx, ops, bad, bf16):
    if bf16 and np.isfinite(bad):
        bad = float(from_bf16(np.array([0x7F7F], dtype=np.uint16))[0])  # bf16's largest
    for lens, reach in ([0, 1, 19, 200, 33], None), ([64, 7, 130, 1, 0], 40):
        rng = np.random.default_rng(9)
        pool = Pool(slm, ctx, ops, rng, lens, 2, 64, 24, bf16, bad=bad)
        q = rng.standard_normal((len(lens), 4, 64)).astype(np.float32)
        y, tol, drawn = pool.formula(q, 4, 0.125, reach)
        if reach:  # slots before the window are not visible either
            for i, n in enumerate(lens):
                s = np.arange(0, max(0, n - reach))
                for x in (pool.k, pool.v):
                    x[np.asarray(pool.ids[i], dtype=int)[s // 24], :, s % 24] = bad
            pool.kb, pool.vb = pool.up(pool.k), pool.up(pool.v)
        got = pool.attend(ops.upload(q), 4, 0.125, reach, weights=True)
        assert (abs(got - y) <= tol).all()
        np.testing.assert_array_equal(got[np.array(lens) == 0], 0)


def test_attend_reads_strided_queries_and_leaves_the_rest_of_y(slm, ctx, ops):
    rng = np.random.default_rng(11)
    pool = Pool(slm, ctx, ops, rng, [40, 0, 300], 2, 64, 16, False)
    wide = rng.standard_normal((3, 401)).astype(np.float32)  # an odd row stride, an odd offset
    q = wide[:, 5:5 + 256].reshape(3, 4, 64)
    y, tol, _ = pool.formula(q, 4, 0.125)
    out = ops.upload(np.full(3 * 256 + 64, 5.0, dtype=np.float32))
    got = pool.attend((ops.upload(wide), 5), 4, 0.125, ldq=401, y=out)
    assert (abs(got - y) <= tol).all()
    np.testing.assert_array_equal(out.read()[3 * 256:], 5.0)


def test_attend_follows_the_table_in_stream_order(slm, ctx, ops):
    """Lengths and pages set between calls that are still queued; few changes and many."""
    rng = np.random.default_rng(12)
    n, page = 40, 4
    pool = Pool(slm, ctx, ops, rng, [400] * n, 1, 32, page, False)
    q = rng.standard_normal((n, 2, 32)).astype(np.float32)
    qb, outs = ops.upload(q), []
    scores = [ops.zeros(1) for _ in range(5)]
    for step in range(5):
        lens = [(37 * i + 90 * step) % 401 for i in range(n)]
        pool.table.set_lens([0] * n)
        for i in range(n):  # 4000 page ids change where the order of the pages turns round
            pool.table.assign(i, pool.ids[i][::-1] if step == 3 else pool.ids[i])
        pool.table.set_lens(lens)
        outs.append((lens, step, ops.zeros(1)))
        ops.paged_attend(outs[-1][2], scores[step], qb, pool.kb, pool.vb, pool.table, heads=2, key_heads=1, dh=32,
                         scale=0.2)
    plain = [list(r) for r in pool.ids]
    for lens, step, y in outs:
        pool.lens, pool.ids = lens, [r[::-1] if step == 3 else r for r in plain]
        want, tol, _ = pool.formula(q, 2, 0.2)
        assert (abs(y.read().reshape(n, 2, 32) - want) <= tol).all()
    np.testing.assert_array_equal(pool.table.lens(), outs[-1][0])


@pytest.mark.parametrize("weights", [False, True])
def test_scratch_of_a_decode_loop_grows_by_a_quarter_at_least(slm, ctx, ops, weights):
    """A step that needs more scratch waits for it, so steps that follow are to find some left."""
    rng = np.random.default_rng(31)
    pool = Pool(slm, ctx, ops, rng, [640, 500], 2, 64, 16, False)
    q = rng.standard_normal((2, 6, 64)).astype(np.float32)
    qb, y, scores, sizes = ops.upload(q), ops.zeros(1), ops.zeros(1), []
    for step in range(401):
        pool.table.set_lens([240 + step, 100 + step])
        ops.paged_attend(y, scores, qb, pool.kb, pool.vb, pool.table, heads=6, key_heads=2, dh=64, scale=0.125,
                         weights=pool.wb if weights else None)
        if len(scores) != (sizes or [1])[-1]:
            sizes.append(len(scores))
    assert len(sizes) > 1 and all(4 * b >= 5 * a for a, b in zip(sizes, sizes[1:]))
    want, tol, _ = pool.formula(q, 6, 0.125)
    assert (abs(y.read().reshape(2, 6, 64) - want) <= tol).all()


def test_two_tables_share_a_common_beginning(slm, ctx, ops):
    rng = np.random.default_rng(13)
    pool = Pool(slm, ctx, ops, rng, [50, 20], 2, 64, 16, True, spare=4)
    pool.table.set_lens([50, 0])
    pool.ids[1] = pool.ids[0][:2] + pool.free[:1]
    pool.table.assign(1, pool.ids[1])
    pool.lens = [50, 40]
    pool.table.set_lens(pool.lens)
    q = rng.standard_normal((2, 2, 64)).astype(np.float32)
    y, tol, _ = pool.formula(q, 2, 0.125)
    assert (abs(pool.attend(ops.upload(q), 2, 0.125) - y) <= tol).all()
    with pytest.raises(slm.SlmError, match="two sequences"):
        pool.attend(ops.upload(q), 2, 0.125, weights=True)
    src = ops.zeros(2 * 9 * 128)
    with pytest.raises(slm.SlmError, match="two sequences"):
        ops.paged_store(pool.kb, pool.vb, pool.table, src, src, m=9, key_heads=2, dh=64, bf16=True)


def test_results_do_not_change_from_call_to_call(slm, ctx, ops):
    rng = np.random.default_rng(14)
    pool = Pool(slm, ctx, ops, rng, [5000, 17, 2500, 0, 1], 2, 64, 16, True)
    q = ops.upload(rng.standard_normal((5, 8, 64)))
    first = pool.attend(q, 8, 0.125, weights=True)
    w = pool.weights()
    for _ in range(5):
        pool.wb = ops.upload(pool.w)
        np.testing.assert_array_equal(pool.attend(q, 8, 0.125, weights=True), first)
        np.testing.assert_array_equal(pool.weights(), w)


@pytest.mark.parametrize("bf16", [False, True])
def test_pages_past_32_bit_offsets(slm, ctx, ops, bf16):
    """Pools of more than 2^31 values whose last pages alone are used."""
    rng = np.random.default_rng(15)
    kh, dh, page = 4, 128, 64
    pages = (1 << 31) // (kh * dh * page) + 40
    floats = pages * kh * dh * page // (2 if bf16 else 1)
    kb, vb, wb = ops.zeros(floats), ops.zeros(floats), ops.zeros(pages * kh * page)
    t = slm.Table(ctx, 1, 8, page, pages)
    t.assign(0, [pages - 1, pages - 3, pages - 30])
    n = 150
    t.set_lens([n])
    k, v = (from_bf16(to_bf16(rng.standard_normal((n, kh, dh)))) for _ in range(2))
    ops.paged_store(kb, vb, t, ops.upload(k), ops.upload(v), m=n, key_heads=kh, dh=dh, bf16=bf16, weights=wb)
    q = rng.standard_normal((kh, dh)).astype(np.float32)
    y, scores = ops.zeros(1), ops.zeros(1)
    args = dict(key_heads=kh, dh=dh, bf16=bf16)
    ops.paged_attend(y, scores, ops.upload(q), kb, vb, t, heads=kh, scale=0.1, weights=wb, **args)
    x = 0.1 * np.einsum("hd,shd->hs", q.astype(np.float64), k)
    p = np.exp(x - x.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    np.testing.assert_allclose(y.read().reshape(kh, dh), np.einsum("hs,shd->hd", p, v), rtol=0, atol=2e-5)
    to = slm.Table(ctx, 1, 8, page, pages)
    to.assign(0, [pages - 20])
    kept = ops.zeros(1)
    ops.paged_evict(kept, kb, vb, wb, t, to, keep=40, sinks=2, recent=10, **args)
    ids = kept.read().view(np.uint32).reshape(kh, 40)
    ops.paged_attend(y, scores, ops.upload(q), kb, vb, to, heads=kh, scale=0.1, **args)
    for h in range(kh):
        ph = p[h, ids[h]] / p[h, ids[h]].sum()
        np.testing.assert_allclose(y.read().reshape(kh, dh)[h], ph @ v[ids[h], h], rtol=0, atol=2e-5)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("lens,kh,dh,page,m,first,count", [
    ([1], 1, 8, 1, 1, 0, 1), ([5, 0, 17, 16], 3, 40, 16, 1, 0, 4), ([5, 0, 17, 16], 4, 64, 16, 7, 0, 4),
    ([700, 3], 8, 128, 32, 700, 0, 2), ([30, 31, 32], 2, 256, 5, 9, 1, 2), ([30, 31, 32], 1, 24, 64, 0, 0, 3),
    ([9, 9], 2, 64, 4, 9, 1, 0)])
def test_store(slm, ctx, ops, bf16, lens, kh, dh, page, m, first, count):
    rng = np.random.default_rng(20)
    pool = Pool(slm, ctx, ops, rng, lens, kh, dh, page, bf16)
    width = kh * dh
    src = rng.standard_normal((max(1, count * m), 2 * width + 3)).astype(np.float32)
    src[0, :4] = [0.0, -0.0, 1.00390625, 3.0e38]  # a tie, and a value near the types' largest
    buf = ops.upload(src)
    ops.paged_store(pool.kb, pool.vb, pool.table, buf, (buf, width + 1), m=m, key_heads=kh, dh=dh, first=first,
                    count=count, ldk=2 * width + 3, ldv=2 * width + 3, bf16=bf16, weights=pool.wb)
    for i in range(first, first + count):
        for j in range(m):
            s = lens[i] - m + j
            if s < 0:
                continue
            page_id, row = pool.ids[i][s // page], s % page
            for x, at in (pool.k, 0), (pool.v, width + 1):
                new = src[(i - first) * m + j, at:at + width].reshape(kh, dh)
                x[page_id, :, row] = from_bf16(to_bf16(new)) if bf16 else new
            pool.w[page_id, :, row] = 0
    np.testing.assert_array_equal(pool.down(pool.kb), pool.k)
    np.testing.assert_array_equal(pool.down(pool.vb), pool.v)
    np.testing.assert_array_equal(pool.weights(), pool.w)


def test_store_keeps_special_values(slm, ctx, ops):
    for bf16 in (False, True):
        pool = Pool(slm, ctx, ops, np.random.default_rng(21), [3], 1, 8, 4, bf16)
        src = np.array([np.inf, -np.inf, np.nan, 3.4e38, 1e-45, -1e-40, 65536.0, -0.0], dtype=np.float32)
        ops.paged_store(pool.kb, pool.vb, pool.table, ops.upload(src), ops.upload(src), m=1, key_heads=1, dh=8, bf16=bf16)
        got = pool.down(pool.vb)[pool.ids[0][0], 0, 2]
        want = src.copy()
        if bf16:
            want[3], want[4:6] = np.inf, from_bf16(to_bf16(src[4:6]))
        np.testing.assert_array_equal(got, want)


def keep_slots(w, n, keep, sinks, recent):
    """The kept slots of one key head by the rule, w its weights."""
    if n <= keep:
        return np.arange(n)
    held = list(range(sinks)) + list(range(n - recent, n))
    order = sorted(range(sinks, n - recent), key=lambda s: (np.isnan(w[s]), 0.0 if np.isnan(w[s]) else -float(w[s]), s))
    return np.sort(held + order[: keep - len(held)])


EVICT = [
    # lens, key_heads, dh, page, bf16, keep, sinks, recent, weights
    ([1], 1, 8, 1, False, 1, 0, 0, "random"),
    ([2, 1, 0], 1, 8, 1, False, 1, 0, 0, "random"),
    ([40, 0, 300, 17], 2, 64, 16, True, 32, 4, 8, "random"),
    ([40, 0, 300, 17], 3, 40, 24, False, 32, 32, 0, "random"),
    ([40, 0, 300, 17], 3, 40, 24, False, 32, 0, 32, "random"),
    ([1000, 999], 2, 64, 16, True, 999, 1, 1, "random"),
    ([2048, 2047, 1025], 4, 64, 64, False, 1024, 4, 256, "ties"),
    ([2048, 1500], 2, 128, 32, True, 700, 4, 64, "equal"),
    ([2048, 1500], 2, 64, 32, True, 700, 0, 0, "special"),
    ([9000, 20, 5000], 2, 32, 16, True, 4097, 4, 1000, "random"),
    ([70000], 2, 16, 64, True, 20001, 4, 100, "ties"),
    ([300], 1, 256, 7, False, 20, 1, 2, "tiny"),
    ([(i * 97) % 1300 for i in range(40)], 3, 24, 16, True, 500, 2, 64, "random"),
    ([(i * 97) % 1300 for i in range(40)], 4, 64, 8, False, 500, 0, 0, "ties"),
    ([500000], 1, 8, 256, True, 70000, 4, 100, "random"),
]


@pytest.mark.parametrize("case", range(len(EVICT)))
def test_evict(slm, ctx, ops, case):
    lens, kh, dh, page, bf16, keep, sinks, recent, kind = EVICT[case]
    rng = np.random.default_rng(300 + case)
    to_per = max(1, -(-min(max(lens), keep) // page))
    pool = Pool(slm, ctx, ops, rng, lens, kh, dh, page, bf16, spare=len(lens) * to_per + 2)
    if kind == "ties":
        pool.w = rng.integers(0, 6, pool.w.shape).astype(np.float32) / 4
    elif kind == "equal":
        pool.w[:] = 0.25
    elif kind == "special":
        pick = rng.integers(0, 7, pool.w.shape)
        for j, x in enumerate([0.0, -0.0, np.nan, np.inf, -1.0, 1e-42, -np.inf]):
            pool.w[pick == j] = x
    elif kind == "tiny":
        pool.w = (rng.integers(0, 1 << 12, pool.w.shape).astype(np.uint32)).view(np.float32)  # subnormals
    pool.wb = ops.upload(pool.w)
    to = slm.Table(ctx, len(lens), to_per, page, pool.pages)
    to_ids = [pool.free[i * to_per:(i + 1) * to_per] for i in range(len(lens))]
    for i, ids in enumerate(to_ids):
        to.assign(i, ids)
    kept = ops.zeros(len(lens) * kh * keep)
    for _ in range(2):  # the pages it reads stay: a second call does the same
        ops.paged_evict(kept, pool.kb, pool.vb, pool.wb, pool.table, to, keep=keep, sinks=sinks, recent=recent,
                        key_heads=kh, dh=dh, bf16=bf16)
    got = kept.read()[: len(lens) * kh * keep].view(np.uint32).reshape(len(lens), kh, keep)
    k, v, w = pool.k.copy(), pool.v.copy(), pool.w.copy()
    for i, n in enumerate(lens):
        for h in range(kh):
            ws = pool.rows(pool.w, i, 0, n)[h] if n else np.zeros(0, np.float32)
            old = keep_slots(ws, n, keep, sinks, recent)
            np.testing.assert_array_equal(got[i, h, :len(old)], old)
            assert (got[i, h, len(old):] == 0xFFFFFFFF).all()
            new = np.arange(len(old))
            if not len(old):
                continue
            a = np.asarray(pool.ids[i])[old // page], h, old % page
            b = np.asarray(to_ids[i])[new // page], h, new % page
            k[b], v[b], w[b] = pool.k[a], pool.v[a], pool.w[a]
    np.testing.assert_array_equal(pool.down(pool.kb), k)
    np.testing.assert_array_equal(pool.down(pool.vb), v)
    np.testing.assert_array_equal(pool.weights(), w)
    np.testing.assert_array_equal(to.lens(), np.minimum(lens, keep))
    np.testing.assert_array_equal(pool.table.lens(), lens)


@pytest.mark.parametrize("bf16", [False, True])
def test_a_decode_loop_with_a_budget(slm, ctx, ops, bf16):
    """Prompts stored at once, then tokens one by one: store, attend with weights, and an eviction to other
    pages whenever the longest cache passes the budget by 16, against the formulas in 64 bits.  Which tokens an
    eviction keeps is taken from the device (nearly equal weights may fall either way) and checked by weight."""
    rng = np.random.default_rng(40)
    n, heads, kh, dh, page, budget, steps = 3, 6, 2, 64, 8, 48, 40
    args = dict(key_heads=kh, dh=dh, bf16=bf16)
    per = (budget + 16 + page - 1) // page
    pages = 2 * n * per
    floats = pages * kh * page * dh // (2 if bf16 else 1)
    kb, vb, wb = ops.zeros(floats), ops.zeros(floats), ops.zeros(pages * kh * page)
    tables = [slm.Table(ctx, n, per, page, pages) for _ in range(2)]
    order = rng.permutation(pages).reshape(2, n, per)
    for t, ids in zip(tables, order):
        for i in range(n):
            t.assign(i, ids[i])
    lens = [30, 0, 61]  # the middle sequence joins later
    hold = (lambda x: from_bf16(to_bf16(x))) if bf16 else (lambda x: x)
    cache = [[[] for _ in range(kh)] for _ in range(n)]  # per key head: [k, v, weight]
    y, scores, kept = ops.zeros(1), ops.zeros(1), ops.zeros(1)
    evictions = 0

    def put(i, new_k, new_v):
        for h in range(kh):
            cache[i][h].append([hold(new_k[h]).astype(np.float64), hold(new_v[h]).astype(np.float64), 0.0])

    for i in range(n):
        if lens[i]:
            k, v = rng.standard_normal((2, lens[i], kh, dh)).astype(np.float32)
            tables[0].set_lens([lens[j] if j <= i else 0 for j in range(n)])
            ops.paged_store(kb, vb, tables[0], ops.upload(k), ops.upload(v), m=lens[i], first=i, count=1, weights=wb,
                            **args)
            for a, b in zip(k, v):
                put(i, a, b)
    for step in range(steps):
        if step >= 5:
            lens[1] += 1
        lens[0], lens[2] = lens[0] + 1, lens[2] + 1
        qkv = rng.standard_normal((n, (heads + 2 * kh) * dh)).astype(np.float32)
        buf, ld = ops.upload(qkv), qkv.shape[1]
        tables[0].set_lens(lens)
        ops.paged_store(kb, vb, tables[0], (buf, heads * dh), (buf, (heads + kh) * dh), m=1, ldk=ld, ldv=ld, weights=wb,
                        **args)
        ops.paged_attend(y, scores, buf, kb, vb, tables[0], heads=heads, scale=0.125, ldq=ld, weights=wb, **args)
        got = y.read(n * heads * dh).reshape(n, heads, dh)
        for i in range(n):
            if lens[i] == 0:
                np.testing.assert_array_equal(got[i], 0)
                continue
            new = qkv[i, heads * dh:].reshape(2, kh, dh)
            put(i, new[0], new[1])
            for h in range(kh):
                k, v = (np.array([c[j] for c in cache[i][h]]) for j in (0, 1))
                q = qkv[i, :heads * dh].reshape(heads, dh)[h * 3:h * 3 + 3].astype(np.float64)
                p = np.exp(0.125 * q @ k.T)
                p /= p.sum(-1, keepdims=True)
                # Scores of size ~10 at most: 2e-5 is 100 roundings of them, as in Pool.formula.
                np.testing.assert_allclose(got[i, h * 3:h * 3 + 3], p @ v, rtol=0, atol=1e-4)
                for c, drawn in zip(cache[i][h], p.sum(0)):
                    c[2] += drawn
        if max(lens) >= budget + 16:
            evictions += 1
            ops.paged_evict(kept, kb, vb, wb, tables[0], tables[1], keep=budget, sinks=2, recent=8, **args)
            ids = kept.read(n * kh * budget).view(np.uint32).reshape(n, kh, budget)
            for i in range(n):
                count = min(lens[i], budget)
                for h in range(kh):
                    slots = ids[i, h, :count].tolist()
                    w = np.array([c[2] for c in cache[i][h]])
                    gone = sorted(set(range(lens[i])) - set(slots))
                    assert len(set(slots)) == count and slots == sorted(slots)
                    if gone:
                        middle = [s for s in slots if 2 <= s < lens[i] - 8]
                        assert w[middle].min() >= w[gone].max() * (1 - 1e-4)
                        assert set(range(2)) | set(range(lens[i] - 8, lens[i])) <= set(slots)
                    cache[i][h] = [cache[i][h][s] for s in slots]
                lens[i] = count
            tables.reverse()
            np.testing.assert_array_equal(tables[0].lens(), lens)
    assert evictions >= 2


@pytest.mark.parametrize("bf16", [False, True])
def test_queued_calls_do_as_calls_one_by_one(slm, ctx, ops, bf16):
    """Kernels begin before their predecessors end: a queue of stores, attentions, table changes, other
    operators and evictions gives the bits of the same calls with a wait after each."""
    n, heads, kh, dh, page, per = 5, 8, 2, 64, 4, 40
    pages = 2 * n * per
    floats = pages * kh * page * dh // (2 if bf16 else 1)
    args = dict(key_heads=kh, dh=dh, bf16=bf16)
    results = []
    for wait in (True, False):
        rng = np.random.default_rng(44)
        done = ctx.sync if wait else (lambda: None)
        kb, vb, wb = ops.zeros(floats), ops.zeros(floats), ops.zeros(pages * kh * page)
        tables = [slm.Table(ctx, n, per, page, pages) for _ in range(2)]
        order = rng.permutation(pages).reshape(2, n, per)
        for t, ids in zip(tables, order):
            for i in range(n):
                t.assign(i, ids[i])
        lens = [100, 7, 0, 130, 64]
        src = [ops.upload(rng.standard_normal(n * (heads + 2 * kh) * dh)) for _ in range(4)]
        y, out, scores, kept = ops.zeros(n * heads * dh), ops.zeros(n * heads * dh), ops.zeros(1), ops.zeros(1)
        ld = (heads + 2 * kh) * dh
        for step in range(60):
            lens = [v + (v < per * page) for v in lens]
            tables[0].set_lens(lens)
            ops.paged_store(kb, vb, tables[0], (src[step % 4], heads * dh), (src[step % 4], (heads + kh) * dh), m=1,
                            ldk=ld, ldv=ld, weights=wb, **args)
            done()
            ops.paged_attend(y, scores, src[(step + 1) % 4], kb, vb, tables[0], heads=heads, scale=0.125, ldq=ld,
                             weights=wb if step % 2 else None, **args)
            done()
            ops.add(out, out, y, n * heads * dh)
            done()
            if step % 7 == 6:
                ops.paged_evict(kept, kb, vb, wb, tables[0], tables[1], keep=90, sinks=1, recent=8, **args)
                done()
                tables.reverse()
                lens = [min(v, 90) for v in lens]
        results.append([b.read() for b in (kb, vb, wb, y, out, kept)])
    for a, b in zip(*results):
        np.testing.assert_array_equal(a.view(np.uint32), b.view(np.uint32))


def test_two_contexts_at_once(slm, ctx, ops):
    """Each context has its stream, scratch and counters: calls of two of them overlap on the GPU."""
    rng = np.random.default_rng(41)
    other = slm.Context(0)
    pools = [Pool(slm, c, slm.Ops(c), rng, [3000, 1, 2000], 2, 64, 16, True) for c in (ctx, other)]
    q = rng.standard_normal((3, 8, 64)).astype(np.float32)
    runs = []
    for p in pools:
        runs.append([(p.ops.upload(q), p.ops.zeros(1), p.ops.zeros(1)) for _ in range(4)])
    for a in zip(*runs):
        for p, (qb, y, scores) in zip(pools, a):
            p.ops.paged_attend(y, scores, qb, p.kb, p.vb, p.table, heads=8, key_heads=2, dh=64, scale=0.125, bf16=True)
    for p, made in zip(pools, runs):
        want, tol, _ = p.formula(q, 8, 0.125)
        for _, y, _ in made:
            assert (abs(y.read().reshape(3, 8, 64) - want) <= tol).all()


def test_refusals(slm, ctx, ops):
    import gc

    import torch
    rng = np.random.default_rng(42)
    pool = Pool(slm, ctx, ops, rng, [20, 3], 2, 64, 16, False)
    q, y, scores = ops.zeros(2 * 4 * 64), ops.zeros(1), ops.zeros(1)
    good = dict(heads=4, key_heads=2, dh=64, scale=0.125)

    def attend(y=y, scores=scores, q=q, k=pool.kb, v=pool.vb, table=pool.table, ops=ops, **more):
        ops.paged_attend(y, scores, q, k, v, table, **{**good, **more})

    def refused(call, *args, **more):
        with pytest.raises(slm.SlmError) as e:
            call(*args, **more)
        assert e.value.code == 1, e.value
    attend()
    for more in (dict(heads=3), dict(heads=0), dict(key_heads=0), dict(dh=60), dict(dh=0), dict(dh=264), dict(reach=0),
                 dict(ldq=255), dict(q=(q, 1)), dict(q=ops.zeros(511)), dict(k=ops.zeros(100)), dict(v=ops.zeros(100)),
                 dict(weights=ops.zeros(10)), dict(key_heads=4), dict(k=pool.vb), dict(y=q), dict(scores=y),
                 dict(key_heads=1 << 62, heads=1 << 62), dict(ldq=1 << 62), dict(weights=pool.kb)):
        refused(attend, **more)
    other = slm.Context(0)
    oops = slm.Ops(other)
    refused(attend, ops=oops)
    refused(attend, q=oops.zeros(512))
    refused(attend, table=slm.Table(other, 2, 4, 16, pool.pages))
    src = ops.zeros(2 * 128)
    put = dict(m=1, key_heads=2, dh=64)
    ops.paged_store(pool.kb, pool.vb, pool.table, src, src, **put)
    for more in (dict(m=2), dict(ldk=127), dict(first=3), dict(first=1, count=2), dict(dh=12), dict(m=1 << 40),
                 dict(bf16=True, dh=4)):
        refused(ops.paged_store, pool.kb, pool.vb, pool.table, src, src, **{**put, **more})
    refused(ops.paged_store, pool.kb, pool.vb, pool.table, pool.kb, src, **put)
    refused(ops.paged_store, pool.kb, pool.kb, pool.table, src, src, **put)
    refused(ops.paged_store, pool.kb, pool.vb, pool.table, (src, 1), src, **put)
    to = slm.Table(ctx, 2, 2, 16, pool.pages)
    kept = ops.zeros(1)
    cut = dict(keep=4, sinks=1, recent=1, key_heads=2, dh=64)
    refused(ops.paged_evict, kept, pool.kb, pool.vb, pool.wb, pool.table, to, **cut)  # no pages to go to
    to.assign(0, pool.free[:1])
    to.assign(1, pool.free[1:2])
    for more in (dict(keep=0), dict(sinks=4), dict(recent=4), dict(keep=17), dict(dh=7)):
        refused(ops.paged_evict, kept, pool.kb, pool.vb, pool.wb, pool.table, to, **{**cut, **more})
    refused(ops.paged_evict, pool.wb, pool.kb, pool.vb, pool.wb, pool.table, to, **cut)
    refused(ops.paged_evict, kept, pool.kb, pool.vb, pool.wb, pool.table, pool.table, **cut)
    np.testing.assert_array_equal(to.lens(), 0)
    ops.paged_evict(kept, pool.kb, pool.vb, pool.wb, pool.table, to, **cut)
    np.testing.assert_array_equal(to.lens(), [4, 3])
    refused(pool.table.assign, 0, [pool.pages])
    refused(pool.table.set_lens, [33, 0])
    # A capture of the context's stream: refused, and the capture stays usable.
    ctx.sync()
    g = torch.cuda.CUDAGraph()
    stream = torch.cuda.ExternalStream(ctx.stream)
    x = torch.zeros(8, device="cuda")
    x += 1  # its kernel is loaded before the capture
    x.zero_()
    torch.cuda.synchronize()
    gc.collect()
    gc.disable()  # a buffer freed during the capture would wait for the stream
    try:
        with torch.cuda.graph(g, stream=stream, capture_error_mode="thread_local"):
            x += 1
            refused(attend)
            refused(ops.paged_store, pool.kb, pool.vb, pool.table, src, src, **put)
            refused(ops.paged_evict, kept, pool.kb, pool.vb, pool.wb, pool.table, to, **cut)
    finally:
        gc.enable()
    g.replay()
    torch.cuda.synchronize()
    assert x.tolist() == [1.0] * 8
    attend()
    ctx.sync()


def evicted(slm, ctx, ops, pool, keep, sinks, recent):
    """An eviction of the whole pool's sequences, checked whole: kept slots, K, V, weights, lengths."""
    lens, kh, page = pool.lens, pool.kh, pool.page
    to_per = max(1, -(-min(max(lens), keep) // page))
    to = slm.Table(ctx, len(lens), to_per, page, pool.pages)
    to_ids = [pool.free[i * to_per:(i + 1) * to_per] for i in range(len(lens))]
    for i, ids in enumerate(to_ids):
        to.assign(i, ids)
    kept = ops.zeros(len(lens) * kh * keep)
    ops.paged_evict(kept, pool.kb, pool.vb, pool.wb, pool.table, to, keep=keep, sinks=sinks, recent=recent,
                    key_heads=kh, dh=pool.dh, bf16=pool.bf16)
    got = kept.read().view(np.uint32).reshape(len(lens), kh, keep)
    k, v, w = pool.k.copy(), pool.v.copy(), pool.w.copy()
    for i, n in enumerate(lens):
        for h in range(kh):
            ws = pool.rows(pool.w, i, 0, n)[h] if n else np.zeros(0, np.float32)
            old = keep_slots(ws, n, keep, sinks, recent)
            np.testing.assert_array_equal(got[i, h, :len(old)], old)
            assert (got[i, h, len(old):] == 0xFFFFFFFF).all()
            new = np.arange(len(old))
            if len(old):
                a = np.asarray(pool.ids[i])[old // page], h, old % page
                b = np.asarray(to_ids[i])[new // page], h, new % page
                k[b], v[b], w[b] = pool.k[a], pool.v[a], pool.w[a]
    np.testing.assert_array_equal(pool.down(pool.kb), k)
    np.testing.assert_array_equal(pool.down(pool.vb), v)
    np.testing.assert_array_equal(pool.weights(), w)
    np.testing.assert_array_equal(to.lens(), np.minimum(lens, keep))


# A CTA a pair (short sequences; many pairs), and clusters.
@pytest.mark.parametrize("lens,kh,keep,sinks,recent", [
    ([300, 0, 17, 299], 2, 20, 2, 10), ([600, 1024, 513], 4, 512, 1, 64), ([300, 21], 1, 20, 0, 0),
    ([(i * 97) % 1300 for i in range(100)], 3, 200, 4, 64), ([1500, 400, 3000], 2, 300, 4, 32), ([9000], 2, 500, 2, 100)])
@pytest.mark.parametrize("large", [np.inf, np.finfo(np.float32).max, 2.0 ** 127])
@pytest.mark.parametrize("share", [0.01, 0.2, 1.0])
def test_evict_by_large_weights(slm, ctx, ops, lens, kh, keep, sinks, recent, large, share):
    """Tokens pinned by +inf, and weights up to the largest: fewer, as many, more of them than places."""
    rng = np.random.default_rng(50)
    page = 16
    pool = Pool(slm, ctx, ops, rng, lens, kh, 16, page, False, spare=len(lens) * -(-keep // page) + 1)
    pool.w[rng.random(pool.w.shape) < share] = large
    pool.wb = ops.upload(pool.w)
    evicted(slm, ctx, ops, pool, keep, sinks, recent)


def test_evict_at_the_largest_budget(slm, ctx, ops):
    """2^31 - 1 words of kept: the step after the last would pass 2^31."""
    import torch
    pool = Pool(slm, ctx, ops, np.random.default_rng(51), [5], 1, 8, 4, False)
    to = slm.Table(ctx, 1, 2, 4, pool.pages)
    to.assign(0, pool.free[:2])
    kept, keep = ops.zeros(1), (1 << 31) - 1
    ops.paged_evict(kept, pool.kb, pool.vb, pool.wb, pool.table, to, keep=keep, sinks=0, recent=0, key_heads=1, dh=8)
    ctx.sync()

    class Words:
        __cuda_array_interface__ = {"shape": (keep,), "typestr": "<i4", "data": (kept.ptr, False), "version": 2}
    got = torch.as_tensor(Words(), device="cuda")
    assert got[:6].tolist() == [0, 1, 2, 3, 4, -1]
    assert all(bool((part == -1).all()) for part in got[5:].split(1 << 28))
    np.testing.assert_array_equal(to.lens(), [5])


@pytest.mark.parametrize("mode", ["relaxed", "thread_local"])
def test_tables_are_neither_made_nor_freed_in_a_capture(slm, ctx, ops, mode):
    """Both are refused, the capture stays usable, and the tables are as they were."""
    import gc

    import torch
    rng = np.random.default_rng(52)
    pool = Pool(slm, ctx, ops, rng, [20, 3], 2, 64, 16, False)
    q = rng.standard_normal((2, 4, 64)).astype(np.float32)
    qb = ops.upload(q)
    stream, g = torch.cuda.ExternalStream(ctx.stream), torch.cuda.CUDAGraph()
    x = torch.zeros(8, device="cuda")
    x += 1
    x.zero_()
    ctx.sync()
    torch.cuda.synchronize()
    gc.collect()
    gc.disable()  # a buffer freed during the capture would wait for the stream
    try:
        with torch.cuda.graph(g, stream=stream, capture_error_mode=mode):
            x += 1
            with pytest.raises(slm.SlmError, match="captured") as e:
                slm.Table(ctx, 2, 4, 16, 64)
            pool.table.close()
            pool.table.set_lens([19, 4])
    finally:
        gc.enable()
    assert e.value.code == 1
    g.replay()
    torch.cuda.synchronize()
    assert x.tolist() == [1.0] * 8
    pool.lens = [19, 4]
    np.testing.assert_array_equal(pool.table.lens(), pool.lens)
    y, tol, _ = pool.formula(q, 4, 0.125)
    assert (abs(pool.attend(qb, 4, 0.125) - y) <= tol).all()
    slm.Table(ctx, 2, 4, 16, 64).close()
    pool.table.close()
    assert pool.table._h is None


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("value,key", [(2.0 ** 106, 2.0 ** 60), (2.0 ** -60, 2.0 ** -60), (1.0, 2.0 ** 120)])
def test_attend_with_large_and_small_values(slm, ctx, ops, bf16, value, key):
    """Values up to 2^119 / visible tokens, and keys and queries whose sizes make up for one another."""
    rng = np.random.default_rng(53)
    pool = Pool(slm, ctx, ops, rng, [1000, 9], 2, 64, 16, bf16)
    pool.k, pool.v = pool.k * np.float32(key), np.clip(pool.v, -4, 4) * np.float32(value)
    pool.kb, pool.vb = pool.up(pool.k), pool.up(pool.v)
    q = (rng.standard_normal((2, 6, 64)) / key).astype(np.float32)
    y, tol, drawn = pool.formula(q, 6, 0.125)
    got = pool.attend(ops.upload(q), 6, 0.125, weights=True)
    assert (abs(got - y) <= tol).all(), float((abs(got - y) / tol).max())
    pool.check_weights(pool.w, pool.weights(), drawn)


def test_evicting_from_a_common_beginning(slm, ctx, ops):
    """Two sequences that list the same first pages go to pages of their own; the shared ones stay."""
    rng = np.random.default_rng(54)
    pool = Pool(slm, ctx, ops, rng, [50, 40], 2, 64, 16, True, spare=8)
    pool.table.set_lens([50, 0])
    pool.ids[1] = pool.ids[0][:2] + pool.ids[1][2:]
    pool.table.assign(1, pool.ids[1])
    pool.table.set_lens(pool.lens)
    evicted(slm, ctx, ops, pool, 24, 2, 8)
