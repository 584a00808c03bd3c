"""The paged key-value cache on the GPU: append, attention of one new token, eviction by
accumulated weight, against the definitions in 64 bits (tests/decoder_cases.py, which derives
the tolerances).  Places that no row fills hold NaN, and so do hidden ones."""
import numpy as np
import pytest

from tests import decoder_cases as dc

pytestmark = pytest.mark.gpu


@pytest.fixture
def tf(cuda_engine):
    from tfjs_b200 import ops
    backend = cuda_engine.backend
    before = backend.numDataIds()
    yield ops
    backend.sync()
    assert backend.numDataIds() == before


class Held(object):
    """Tensors of a cache, disposed together."""

    def __init__(self, tf, cache, lengths=None):
        self.tf, self.all = tf, []
        self.k, self.v = self(cache.k), self(cache.v)
        self.table = self(cache.table)
        self.lengths = self(cache.lengths if lengths is None else lengths)

    def __call__(self, x):
        if x is None:
            return None
        t = x if hasattr(x, "dataId") else self.tf.tensor(x)
        self.all.append(t)
        return t

    def close(self):
        for t in self.all:
            t.dispose()


def check(got, ref, off):
    assert got.shape == ref.shape
    assert np.all(np.abs(got - ref) <= off), (np.max(np.abs(got - ref)), np.max(np.abs(got - ref) / off))


def attend(tf, cache, q, scale=None, mask=None, weights=None):
    h = Held(tf, cache)
    got = tf.paged_attention(h(q), h.k, h.v, h.table, h.lengths, scale, h(mask), h(weights))
    outs = [h(t).arraySync() for t in (got if isinstance(got, list) else [got])]
    h.close()
    return outs


SHAPES = [
    # heads, kv_heads, dim, page, lengths
    (1, 1, 1, 1, [1]),
    (1, 1, 64, 16, [0, 1, 2]),
    (12, 12, 64, 16, [128]),
    (2, 1, 32, 8, [31, 32, 33]),
    (8, 2, 128, 16, [127, 128, 129, 0, 1]),
    (16, 2, 128, 32, [300, 5, 1000]),
    (7, 1, 80, 3, [100, 99, 1]),
    (9, 1, 100, 5, [260]),
    (16, 1, 16, 64, [513, 64]),
    (6, 2, 33, 7, [50, 0, 77]),
    (3, 3, 7, 128, [129, 200]),
    (8, 4, 192, 16, [90, 33]),
    (4, 1, 256, 24, [70, 333]),
    (32, 2, 255, 16, [40]),
    (5, 5, 2, 2, [11, 3]),
    (40, 1, 64, 16, [200, 3]),
    (6, 2, 128, 16, [400, 30]),
    (24, 2, 20, 4, [70, 260, 1]),
    (4, 1, 96, 1, [77]),
]


@pytest.mark.parametrize("heads,kv,dim,page,lengths", SHAPES)
def test_attention(tf, heads, kv, dim, page, lengths):
    r = np.random.default_rng(dim * 31 + heads)
    cache = dc.Cache(dim + heads, kv, dim, page, lengths)
    q = r.standard_normal((len(lengths), heads, 1, dim)).astype(np.float32)
    scale = 1.0 / np.sqrt(dim)
    ref, _, off, _ = dc.attention(q, cache, lengths, scale)
    (got,) = attend(tf, cache, q, scale)
    check(got, ref, off)
    # with a mask that hides some slots, and the accumulated weights
    mask = np.where(r.random((len(lengths), cache.capacity)) < 0.3, -np.inf,
                    r.standard_normal((len(lengths), cache.capacity))).astype(np.float32)
    w = r.random((len(lengths), kv, cache.capacity)).astype(np.float32)
    ref, neww, off, woff = dc.attention(q, cache, lengths, None, mask, w)
    got, gotw = attend(tf, cache, q, None, mask, w)
    check(got, ref, off)
    check(gotw, neww, woff)


def test_attention_of_a_long_row(tf):
    """The row is split over many blocks; a short row next to it fills one of them."""
    r = np.random.default_rng(5)
    lengths = [20011, 3]
    cache = dc.Cache(5, 2, 64, 64, lengths)
    q = r.standard_normal((2, 8, 1, 64)).astype(np.float32)
    w = r.random((2, 2, cache.capacity)).astype(np.float32)
    ref, neww, off, woff = dc.attention(q, cache, lengths, 0.125, None, w)
    got, gotw = attend(tf, cache, q, 0.125, None, w)
    check(got, ref, off)
    check(gotw, neww, woff)


@pytest.mark.parametrize("heads,kv", [(2, 1), (4, 1), (8, 1), (16, 2)])
def test_many_ragged_rows(tf, heads, kv):
    """More rows than a warp has lanes, empty ones among them: every block takes an equal share of
    the tiles, which begins and ends inside rows."""
    r = np.random.default_rng(heads)
    lengths = [int(n) for n in r.integers(0, 700, 75)]
    lengths[10] = lengths[74] = lengths[0] = 0
    lengths[40] = 1500
    cache = dc.Cache(heads, kv, 32, 16, lengths)
    q = r.standard_normal((75, heads, 1, 32)).astype(np.float32)
    w = r.random((75, kv, cache.capacity)).astype(np.float32)
    ref, neww, off, woff = dc.attention(q, cache, lengths, 0.2, None, w)
    got, gotw = attend(tf, cache, q, 0.2, None, w)
    check(got, ref, off)
    check(gotw, neww, woff)


def test_rows_that_attend_to_nothing(tf):
    """No slots, or only hidden ones: zeros, and nothing is added to the weights."""
    lengths = [0, 40, 40]
    cache = dc.Cache(1, 2, 64, 16, lengths)
    q = np.random.default_rng(1).standard_normal((3, 4, 1, 64)).astype(np.float32)
    mask = np.zeros((3, cache.capacity), np.float32)
    mask[1] = -np.inf
    cache.k[cache.table[1, 0], :, 3] = np.nan        # hidden: must not count
    cache.v[cache.table[1, 0], :, 4] = np.inf
    w = np.random.default_rng(2).random((3, 2, cache.capacity)).astype(np.float32)
    got, gotw = attend(tf, cache, q, 0.125, mask, w)
    assert np.all(got[:2] == 0.0) and np.all(np.isfinite(got))
    assert np.all(gotw[0] == 0.0)
    assert np.array_equal(gotw[1, :, :40], w[1, :, :40]) and np.all(gotw[1, :, 40:] == 0.0)
    ref, _, off, _ = dc.attention(q, cache, lengths, 0.125, mask, w)
    check(got, ref, off)


def test_masks_of_the_lowest_value_and_large_scores(tf):
    """A row masked throughout with the lowest float is a softmax of equals; scores of some
    hundred neither overflow nor lose the largest; a NaN in q poisons its own head."""
    lengths = [50, 50, 50]
    cache = dc.Cache(3, 1, 64, 16, lengths)
    q = np.random.default_rng(3).standard_normal((3, 2, 1, 64)).astype(np.float32)
    q[1] *= 40.0
    q[2, 1, 0, 5] = np.nan
    mask = np.zeros((3, cache.capacity), np.float32)
    mask[0] = np.finfo(np.float32).min
    (got,) = attend(tf, cache, q, None, mask)
    # q k is lost beside 3.4e38, so that all scores are equal
    even = cache.rows(cache.v, 0, 50).astype(np.float64).mean(axis=0)[0]
    spread = np.abs(cache.rows(cache.v, 0, 50)).astype(np.float64).mean(axis=0)[0]
    assert np.all(np.abs(got[0, 0] - even) <= spread * 128 * dc.EPS)
    q2 = np.where(np.isnan(q), 0, q)
    ref, _, off, _ = dc.attention(q2, cache, lengths, None, np.where(mask < -1, 0, mask))
    assert np.all(np.abs(got[1] - ref[1]) <= off[1])
    assert np.all(np.isnan(got[2, 0, 1])) and np.all(np.abs(got[2, 0, 0] - ref[2, 0, 0]) <= off[2, 0, 0])


def test_rows_that_share_pages(tf):
    """Two rows may name the same pages (a common beginning) as long as they only read."""
    cache = dc.Cache(8, 2, 32, 8, [40, 40])
    cache.table[1, :3] = cache.table[0, :3]
    q = np.random.default_rng(8).standard_normal((2, 2, 1, 32)).astype(np.float32)
    ref, _, off, _ = dc.attention(q, cache, [40, 40], 0.2)
    (got,) = attend(tf, cache, q, 0.2)
    check(got, ref, off)


@pytest.mark.parametrize("kv,dim,page,lengths,tokens,counts", [
    (1, 1, 1, [0], 1, None),
    (8, 128, 16, [0, 15, 16, 17], 1, None),
    (2, 64, 16, [0, 5, 31], 40, [40, 0, 17]),
    (3, 33, 5, [7, 0], 23, [1, 23]),
    (2, 20, 128, [100, 128], 300, None),
    (12, 256, 8, [3], 9, [9]),
])
def test_append(tf, kv, dim, page, lengths, tokens, counts):
    r = np.random.default_rng(kv * dim)
    cache = dc.Cache(dim, kv, dim, page, lengths, max_pages=-(-(max(lengths) + tokens) // page))
    k = r.standard_normal((len(lengths), kv, tokens, dim)).astype(np.float32)
    v = r.standard_normal((len(lengths), kv, tokens, dim)).astype(np.float32)
    h = Held(tf, cache)
    new = h(tf.paged_cache_append(h.k, h.v, h(k), h(v), h.table, h.lengths,
                                  h(np.array(counts, np.int32)) if counts else None))
    got = new.arraySync(), h.k.arraySync(), h.v.arraySync()
    h.close()
    c = counts or [tokens] * len(lengths)
    for b, n in enumerate(lengths):
        for t in range(c[b]):
            at = cache.table[b, (n + t) // page], slice(None), (n + t) % page
            cache.k[at], cache.v[at] = k[b, :, t], v[b, :, t]
    assert np.array_equal(got[0], np.array(lengths) + np.array(c))
    assert np.array_equal(got[1], cache.k, equal_nan=True)     # places beside them as they were
    assert np.array_equal(got[2], cache.v, equal_nan=True)


def run_evict(tf, cache, w, budget, recent, positions=None, total=None):
    h = Held(tf, cache)
    outs = tf.paged_cache_evict(h.k, h.v, h(w), h.table, h.lengths, budget, recent,
                                h(positions), h(total))
    got = [h(t).arraySync() for t in outs] + [h.k.arraySync(), h.v.arraySync()]
    h.close()
    return got


@pytest.mark.parametrize("kv,dim,page,lengths,budget,recent,order", [
    (1, 4, 4, [1], 1, 0, False),
    (2, 64, 16, [100, 33, 0, 32, 31], 32, 8, False),
    (2, 64, 16, [100, 33, 0, 32, 31], 32, 32, True),
    (1, 33, 5, [77, 200], 1, 0, False),
    (1, 33, 5, [77, 200], 1, 1, True),
    (8, 128, 16, [1025, 1025], 1024, 256, True),
    (2, 16, 64, [3000, 1023, 1024, 2049], 1024, 100, True),
    (1, 8, 16, [50], 4000, 10, False),
    (3, 24, 8, [500, 17], 250, 0, True),
    (1, 4, 64, [60000, 20], 20000, 7000, True),      # keys do not fit shared memory
    (2, 6, 16, [9000, 4097], 4096, 0, False),
])
def test_evict(tf, kv, dim, page, lengths, budget, recent, order):
    r = np.random.default_rng(budget + dim)
    cache = dc.Cache(budget, kv, dim, page, lengths)
    shape = (len(lengths), kv, cache.capacity)
    w = np.exp(2 * r.standard_normal(shape)).astype(np.float32)
    w[r.random(shape) < 0.3] = 0.0                       # many equals
    w[r.random(shape) < 0.02] *= -1.0
    w[r.random(shape) < 0.01] = np.inf
    w[r.random(shape) < 0.01] = np.nan
    w[:, :, ::7] *= np.float32(-0.0) if budget == 250 else np.float32(1.0)
    positions = total = None
    if order:
        positions = np.argsort(r.random(shape), axis=-1).astype(np.int32)
        positions[r.random(shape) < 0.2] = -1
        total = (np.array(lengths) + 13).astype(np.int32)
    ref = dc.evict(cache, w, lengths, budget, recent, positions, total)
    got = run_evict(tf, cache, w, budget, recent, positions, total)
    for a, b in zip(got, ref):
        assert a.dtype == b.dtype and np.array_equal(a, b, equal_nan=a.dtype == np.float32)


def test_evict_twice_is_evict(tf):
    """A row within its budget is left alone."""
    r = np.random.default_rng(4)
    cache = dc.Cache(4, 2, 32, 16, [90, 64])
    w = r.random((2, 2, cache.capacity)).astype(np.float32)
    w1, p1, l1, _, cache.k, cache.v = run_evict(tf, cache, w, 64, 16)
    cache.lengths = l1
    w2, p2, l2, kept, k, v = run_evict(tf, cache, w1, 64, 16, p1, np.array([90, 64], np.int32))
    assert np.array_equal(w1, w2) and np.array_equal(p1, p2) and np.array_equal(l1, l2)
    assert np.array_equal(kept, np.broadcast_to(np.arange(64), kept.shape))
    assert np.array_equal(k, cache.k, equal_nan=True) and np.array_equal(v, cache.v, equal_nan=True)


def test_bad_pages_and_lengths_are_reported(tf, cuda_engine):
    """The slots of a page that no pool has are left out, lengths are clamped, and the next
    blocking call says so, once."""
    from tfjs_b200 import _cabi
    backend = cuda_engine.backend
    r = np.random.default_rng(6)
    q = r.standard_normal((2, 2, 1, 32)).astype(np.float32)

    def once(f, word):
        outs = f()
        with pytest.raises(_cabi.CudaError) as e:
            backend.sync()
        assert e.value.code == 1 and word in str(e.value)
        backend.sync()
        return outs

    for bad in (-1, 10 ** 6):
        cache = dc.Cache(6, 2, 32, 8, [40, 20])
        good = cache.table[0, 2]
        cache.table[0, 2] = bad
        h = Held(tf, cache)
        got = once(lambda: h(tf.paged_attention(h(q), h.k, h.v, h.table, h.lengths, 0.2)), "page").arraySync()
        cache.table[0, 2] = good
        mask = np.zeros((2, cache.capacity), np.float32)
        mask[0, 16:24] = -np.inf
        ref, _, off, _ = dc.attention(q, cache, [40, 20], 0.2, mask)
        check(got, ref, off)
        # appending into such a page drops what belongs there and nothing else
        k = r.standard_normal((2, 2, 4, 32)).astype(np.float32)
        lengths = h(np.array([14, 20], np.int32))
        new = once(lambda: h(tf.paged_cache_append(h.k, h.v, h(k), h(k), h.table, lengths)), "page").arraySync()
        want = cache.k.copy()
        want[cache.table[0, 1], :, 6:8] = k[0, :, :2]
        want[cache.table[1, 2], :, 4:8] = k[1]
        assert np.array_equal(new, [18, 24]) and np.array_equal(h.k.arraySync(), want, equal_nan=True)
        # eviction leaves such moves out
        w = r.random((2, 2, cache.capacity)).astype(np.float32)
        outs = once(lambda: [h(t) for t in tf.paged_cache_evict(h.k, h.v, h(w), h.table, h.lengths, 20, 4)], "page")
        assert np.array_equal(outs[2].arraySync(), [20, 20])
        h.close()
    cache = dc.Cache(7, 2, 32, 8, [16, 16])
    h = Held(tf, cache, np.array([-5, 1 << 30], np.int32))
    got = once(lambda: h(tf.paged_attention(h(q), h.k, h.v, h.table, h.lengths, 0.2)), "length").arraySync()
    ref, _, off, _ = dc.attention(q, cache, [0, 16], 0.2)
    check(got, ref, off)
    k = r.standard_normal((2, 2, 3, 32)).astype(np.float32)
    counts = h(np.array([4, 3], np.int32))
    lengths = h(np.array([0, 14], np.int32))
    new = once(lambda: h(tf.paged_cache_append(h.k, h.v, h(k), h(k), h.table, lengths, counts)), "length")
    assert np.array_equal(new.arraySync(), [3, 16])
    h.close()


def test_a_few_steps_of_generation(tf, cuda_engine):
    """Append, attend with the weights kept, evict: the parts together, step by step against
    the definitions."""
    r = np.random.default_rng(11)
    B, H, KV, D, P, budget, recent = 3, 8, 2, 64, 8, 24, 6
    start = [24, 10, 3]
    cache = dc.Cache(11, KV, D, P, start, max_pages=4)
    h = Held(tf, cache)
    lengths, total = h.lengths, np.array(start, np.int32)
    w = np.zeros((B, KV, cache.capacity), np.float32)
    pos = np.full((B, KV, cache.capacity), -1, np.int32)
    tw, tp = h(w), h(pos)
    n = np.array(start, np.int32)
    for step in range(20):
        k, v, q = (r.standard_normal((B, x, 1, D)).astype(np.float32) for x in (KV, KV, H))
        lengths = h(tf.paged_cache_append(h.k, h.v, h(k), h(v), h.table, lengths))
        out, tw = [h(t) for t in tf.paged_attention(h(q), h.k, h.v, h.table, lengths, 0.125, None, tw)]
        for b in range(B):
            at = cache.table[b, n[b] // P], slice(None), n[b] % P
            cache.k[at], cache.v[at] = k[b, :, 0], v[b, :, 0]
        n, total = n + 1, total + 1
        ref, neww, off, woff = dc.attention(q, cache, n, 0.125, None, w)
        check(out.arraySync(), ref, off)
        got_w = tw.arraySync()
        check(got_w, neww, woff + 20 * dc.EPS * neww)
        w = got_w                      # the same bits decide on both sides
        tw, tp, lengths, kept = [h(t) for t in tf.paged_cache_evict(
            h.k, h.v, tw, h.table, lengths, budget, recent, tp, h(total))]
        w, pos, n, want_kept, cache.k, cache.v = dc.evict(cache, w, n, budget, recent, pos, total)
        assert np.array_equal(kept.arraySync(), want_kept)
        assert np.array_equal(tw.arraySync(), w) and np.array_equal(tp.arraySync(), pos)
        assert np.array_equal(lengths.arraySync(), n)
        assert np.array_equal(h.k.arraySync(), cache.k, equal_nan=True)
    h.close()


def test_captured_steps_replay(tf, cuda_engine):
    """A captured step (append, attend, lengths and weights copied back) replays on the pools
    as they are by then; two captured steps and eager calls in between do not disturb each
    other."""
    backend = cuda_engine.backend
    r = np.random.default_rng(12)
    B, H, KV, D, P = 2, 4, 2, 64, 16
    cache = dc.Cache(12, KV, D, P, [20, 60], max_pages=6)
    h = Held(tf, cache)
    k, v = (r.standard_normal((B, KV, 1, D)).astype(np.float32) for _ in range(2))
    q = r.standard_normal((B, H, 1, D)).astype(np.float32)
    tk, tv, tq = h(k), h(v), h(q)
    w = h(np.zeros((B, KV, cache.capacity), np.float32))
    for t in (h.k, h.v, h.table, h.lengths, tk, tv, tq, w):
        backend.device_id(t.dataId)
    eager = h(tf.paged_attention(tq, h.k, h.v, h.table, h.lengths, 0.125)).arraySync()

    def step():
        new = tf.paged_cache_append(h.k, h.v, tk, tv, h.table, h.lengths)
        out, neww = tf.paged_attention(tq, h.k, h.v, h.table, new, 0.125, None, w)
        backend.copy(new.dataId, h.lengths.dataId)
        backend.copy(neww.dataId, w.dataId)
        new.dispose()
        neww.dispose()
        return out

    graphs = []
    for _ in range(2):
        backend.sync()
        backend.capture_begin(64 << 20)
        out = step()
        graphs.append((backend.capture_end(), h(out)))
    weights = np.zeros((B, KV, cache.capacity), np.float32)
    n = np.array([20, 60], np.int32)
    for i in range(5):
        graph, out = graphs[i % 2]
        backend.graph_launch(graph)
        if i == 2:
            h(tf.paged_attention(tq, h.k, h.v, h.table, h.lengths, 0.125)).dataSync()
        for b in range(B):
            at = cache.table[b, n[b] // P], slice(None), n[b] % P
            cache.k[at], cache.v[at] = k[b, :, 0], v[b, :, 0]
        n = n + 1
        ref, weights, off, woff = dc.attention(q, cache, n, 0.125, None, weights)
        # (the lengths' and the weights' host copies are from before the replays)
        check(out.arraySync(), ref, off)
    assert not np.array_equal(eager, out.arraySync())
    backend.sync()
    for graph, _ in graphs:
        backend.graph_destroy(graph)
    h.close()


def test_pools_in_place_and_pending_readers(tf, cuda_engine):
    """What was computed lazily from a pool before an append sees the pool as it was; a small
    pool written from the host is read back as the append left it."""
    cache = dc.Cache(9, 1, 4, 4, [3], max_pages=2)
    assert cache.k.nbytes < 4096
    cache.k[np.isnan(cache.k)] = 0.5
    h = Held(tf, cache)
    k = np.full((1, 1, 1, 4), 7.0, np.float32)
    before = h(tf.add(h.k, h(np.float32(1.0))))
    later = h(tf.mul(before, h(np.float32(2.0))))
    h(tf.paged_cache_append(h.k, h.v, h(k), h(k), h.table, h.lengths))
    assert np.array_equal(later.arraySync(), (cache.k + 1.0) * 2.0)
    assert np.array_equal(before.arraySync(), cache.k + 1.0)
    cache.k[cache.table[0, 0], 0, 3] = 7.0
    assert np.array_equal(h.k.arraySync(), cache.k)
    h.close()


def test_long_pools_pass_32_bits(tf, cuda_engine):
    """Rows whose byte (and element) offsets are above 2^32: the last pages of pools of
    4.6 billion values, of which only the used pages are written."""
    import torch
    KV, D, P = 2, 128, 64
    pages = (1 << 32) // (KV * D * P) + 64
    free, _ = torch.cuda.mem_get_info()
    if free < 2.2 * pages * KV * D * P * 4:
        pytest.skip("not enough device memory")
    pools = [torch.empty((pages, KV, P, D), device="cuda") for _ in range(2)]
    cache = dc.Cache(13, KV, D, P, [150, 64])
    high = np.array([[pages - 1, pages - 2, pages - 40], [pages - 3, -1, -1]], np.int32)
    r = np.random.default_rng(13)
    for b, n in enumerate((150, 64)):
        for i in range(-(-n // P)):
            for pool, src in zip(pools, (cache.k, cache.v)):
                pool[int(high[b, i])] = torch.from_numpy(src[cache.table[b, i]]).cuda()
    torch.cuda.synchronize()
    kc, vc = tf.tensor(pools[0]), tf.tensor(pools[1])
    q = r.standard_normal((2, 4, 1, D)).astype(np.float32)
    k = r.standard_normal((2, KV, 1, D)).astype(np.float32)
    h = Held(tf, cache)
    table, lengths, counts = h(high), h(np.array([150, 63], np.int32)), h(np.array([1, 1], np.int32))
    new = h(tf.paged_cache_append(kc, vc, h(k), h(k), table, lengths, counts))
    at = [(cache.table[0, 150 // P], slice(None), 150 % P), (cache.table[1, 0], slice(None), 63)]
    for b in range(2):
        cache.k[at[b]], cache.v[at[b]] = k[b, :, 0], k[b, :, 0]
    w = np.random.default_rng(1).random((2, KV, 3 * P)).astype(np.float32)
    ref, _, off, _ = dc.attention(q, cache, [151, 64], 0.1)
    check(h(tf.paged_attention(h(q), kc, vc, table, new, 0.1)).arraySync(), ref, off)
    outs = [h(t) for t in tf.paged_cache_evict(kc, vc, h(w), table, new, 70, 10)]
    kept = dc.evict(cache, w, [151, 64], 70, 10)
    assert np.array_equal(outs[3].arraySync(), kept[3])
    for i in range(2):
        assert np.array_equal(pools[0][int(high[0, i])].cpu().numpy(), kept[4][cache.table[0, i]], equal_nan=True)
    h.close()
    kc.dispose()
    vc.dispose()
