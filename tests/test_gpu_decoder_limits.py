"""The decoder's operators where sizes and values reach their limits."""
import numpy as np
import pytest

from tests import decoder_cases as dc
from tests.test_gpu_paged_cache import Held, attend, check, run_evict, tf  # noqa: F401  (tf: a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("slots", [11952, 11968, 12288, 12304, 49152, 49168])
@pytest.mark.parametrize("dim", [8, 6])
def test_evict_around_the_shared_memory_steps(tf, slots, dim):
    """Rows whose keys fill the shared memory that a launch has without asking for more, and what it
    can ask for at most; full rows and short ones in long tables."""
    page = 16
    lengths = [slots, 100] if slots < 20000 else [300, 100]
    cache = dc.Cache(slots + dim, 1, dim, page, lengths, max_pages=slots // page)
    r = np.random.default_rng(slots)
    w = r.random((2, 1, slots)).astype(np.float32)
    ref = dc.evict(cache, w, lengths, 60, 20)
    got = run_evict(tf, cache, w, 60, 20)
    for a, b in zip(got, ref):
        assert a.dtype == b.dtype and np.array_equal(a, b, equal_nan=a.dtype == np.float32)


def test_memory_that_a_call_writes_is_its_own(tf, cuda_engine):
    """Tensors over one piece of memory have ids of their own: two pools in one place, new rows inside a
    pool, or overlapping pools are refused, and neighbours are not."""
    import torch
    from tfjs_b200 import _cabi
    x = torch.zeros(4 * 2 * 8 * 16 * 2, device="cuda")
    n = 4 * 2 * 8 * 16
    torch.cuda.synchronize()

    def view(at, *shape):
        return tf.tensor(x[at:at + int(np.prod(shape))].view(*shape))
    kc, vc = view(0, 4, 2, 8, 16), view(n, 4, 2, 8, 16)
    same, over = view(0, 4, 2, 8, 16), view(n // 2, 4, 2, 8, 16)
    table, lengths = tf.tensor(np.array([[0, 1]], np.int32)), tf.tensor(np.array([3], np.int32))
    k = tf.tensor(np.ones((1, 2, 1, 16), np.float32))
    inside = view(n - 32, 1, 2, 1, 16)
    w = tf.tensor(np.zeros((1, 2, 16), np.float32))
    w_inside = view(n, 1, 2, 16)
    q = tf.tensor(np.ones((1, 2, 1, 16), np.float32))
    for bad in (lambda: tf.paged_cache_append(kc, same, k, k, table, lengths),
                lambda: tf.paged_cache_append(kc, over, k, k, table, lengths),
                lambda: tf.paged_cache_append(kc, vc, inside, k, table, lengths),
                lambda: tf.paged_cache_append(kc, vc, k, inside, table, lengths),
                lambda: tf.paged_cache_evict(kc, over, w, table, lengths, 2),
                lambda: tf.paged_cache_evict(kc, vc, w_inside, table, lengths, 2)):
        with pytest.raises(_cabi.CudaError) as e:
            bad()
        assert e.value.code == 1
    outs = [tf.paged_cache_append(kc, vc, k, k, table, lengths)]
    outs.append(tf.paged_attention(q, kc, vc, table, outs[0]))
    outs.append(tf.paged_attention(q, kc, same, table, outs[0]))     # (nothing is written to the pools)
    for t in outs + [kc, vc, same, over, table, lengths, k, inside, w, w_inside, q]:
        t.dispose()
    assert float(x.sum()) == 2 * 2 * 16


@pytest.mark.parametrize("heads,kv,dim", [(2, 1, 64), (4, 1, 128), (8, 1, 64), (16, 1, 32), (4, 2, 33)])
def test_pages_that_the_mask_hides_are_not_needed(tf, cuda_engine, heads, kv, dim):
    """A window over a long row: the pages in front of it have been given back, their entries name
    none, and the mask hides their slots.  Nothing is wrong with such a call."""
    from tfjs_b200 import _cabi
    page, lengths = 8, [300, 40, 9]
    r = np.random.default_rng(dim)
    cache = dc.Cache(dim, kv, dim, page, lengths)
    mask = np.zeros((3, cache.capacity), np.float32)
    mask[0, :203] = mask[1, :16] = -np.inf
    q = r.standard_normal((3, heads, 1, dim)).astype(np.float32)
    w = r.random((3, kv, cache.capacity)).astype(np.float32)
    ref, neww, off, woff = dc.attention(q, cache, lengths, 0.2, mask, w)
    cache.table[0, :203 // page] = -1
    cache.table[1, :2] = 10 ** 6
    got, gotw = attend(tf, cache, q, 0.2, mask, w)        # (reads block: an error would be raised)
    check(got, ref, off)
    check(gotw, neww, woff)
    # one slot of such a page is shown: reported
    mask[0, 100] = 0.0
    h = Held(tf, cache)
    h(tf.paged_attention(h(q), h.k, h.v, h.table, h.lengths, 0.2, h(mask)))
    with pytest.raises(_cabi.CudaError) as e:
        cuda_engine.backend.sync()
    h.close()
    assert e.value.code == 1 and "page" in str(e.value)


@pytest.mark.parametrize("kv,dim,budget", [(2, 64, 24), (1, 6, 150)])
def test_a_captured_step_that_evicts_replays(tf, cuda_engine, kv, dim, budget):
    """Append, attend with the weights kept, evict, with lengths, weights, positions and totals copied back:
    replayed with eager calls in between, against the definitions; afterwards every state reads as the
    replays left it."""
    backend = cuda_engine.backend
    r = np.random.default_rng(budget)
    B, H, P, recent = 2, 2 * kv, 8, 6
    n = np.array([budget, 5], np.int32)
    cache = dc.Cache(budget, kv, dim, P, n, max_pages=-(-(2 * budget + 90) // P))
    h = Held(tf, cache)
    shape = (B, kv, cache.capacity)
    w, pos = np.zeros(shape, np.float32), np.full(shape, -1, np.int32)
    total = n.copy()
    k, v = (r.standard_normal((B, kv, 1, dim)).astype(np.float32) for _ in range(2))
    q = r.standard_normal((B, H, 1, dim)).astype(np.float32)
    tk, tv, tq, tw, tp, tt, one = (h(x) for x in (k, v, q, w, pos, total, np.ones(1, np.int32)))
    for t in h.all:
        backend.device_id(t.dataId)
    backend.sync()
    backend.capture_begin(64 << 20)
    long = tf.paged_cache_append(h.k, h.v, tk, tv, h.table, h.lengths)
    seen = tf.add(tt, one)
    out, summed = tf.paged_attention(tq, h.k, h.v, h.table, long, 0.25, None, tw)
    parts = tf.paged_cache_evict(h.k, h.v, summed, h.table, long, budget, recent, tp, seen)
    for new, old in zip(parts[:3] + [seen], (tw, tp, h.lengths, tt)):
        backend.copy(new.dataId, old.dataId)
    graph = backend.capture_end()
    h.all += [long, seen, out, summed] + parts
    for step in range(12):
        backend.graph_launch(graph)
        if step % 4 == 3:
            h(tf.paged_attention(tq, h.k, h.v, h.table, h.lengths, 0.25))
        for b in range(B):
            at = cache.table[b, n[b] // P], slice(None), n[b] % P
            cache.k[at], cache.v[at] = k[b, :, 0], v[b, :, 0]
        n, total = n + 1, total + 1
        ref, neww, off, woff = dc.attention(q, cache, n, 0.25, None, w)
        check(out.arraySync(), ref, off)
        got = summed.arraySync()
        check(got, neww, woff + 12 * dc.EPS * neww)
        w, pos, n, kept, cache.k, cache.v = dc.evict(cache, got, n, budget, recent, pos, total)
        assert np.array_equal(parts[3].arraySync(), kept)
    for t, want in ((tw, w), (tp, pos), (h.lengths, n), (tt, total), (h.k, cache.k), (h.v, cache.v)):
        assert np.array_equal(t.arraySync(), want, equal_nan=want.dtype == np.float32)
    backend.graph_destroy(graph)
    h.close()
