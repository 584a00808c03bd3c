"""Device memory that somebody else holds and writes: pending operations, packed weights, order
against streams."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def test_an_upload_that_is_handed_out_at_once(cuda_engine):
    """The holder's stream finds what write_from and the weight loader sent, although no kernel of
    this backend has used it yet."""
    from tfjs_b200 import io
    from tfjs_b200.backend import TensorInfo
    backend = cuda_engine.backend
    before = backend.numDataIds()
    n = 1 << 24
    side = torch.cuda.Stream()
    src = backend.pinned_empty([n], "float32")
    src[:] = np.arange(n, dtype=np.float32)[::-1]

    def summed(t):
        with torch.cuda.stream(side):
            g = torch.as_tensor(t.dataToGPU(side.cuda_stream), device="cuda")
            return g.double().sum().item()
    for _ in range(3):
        src[:n // 2] += np.float32(1.0)                  # (other values each time: blocks are used again)
        dataId = backend.write_from(src, [n], "float32")
        t = cuda_engine.make_tensor_from_info(TensorInfo(dataId, [n], "float32"))
        backend.signal_stream(side.cuda_stream)          # (nothing new for this stream)
        assert summed(t) == src.astype(np.float64).sum()
        t.dispose()
    for _ in range(3):
        src[:n // 2] += np.float32(1.0)
        ws = io.load_weights(cuda_engine, [src.tobytes()], [{"name": "w", "shape": [n], "dtype": "float32"}])
        assert summed(ws["w"]) == src.astype(np.float64).sum()
        ws["w"].dispose()
    assert backend.numDataIds() == before


def test_from_one_stream_through_a_tensor_to_another(cuda_engine):
    """A tensor over memory that stream A fills, handed on to stream B, which was signalled just before:
    B waits for A."""
    from tfjs_b200 import ops as tf
    backend = cuda_engine.backend
    before = backend.numDataIds()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    n = 1 << 25
    x = torch.zeros(n, device="cuda")
    torch.cuda.synchronize()
    for i in range(4):
        for s in (a, b):                     # either has been the one signalled last
            backend.signal_stream(s.cuda_stream)
        with torch.cuda.stream(a):
            for _ in range(50):
                x += 1.0
        t = tf.tensor(x, stream=a.cuda_stream)
        with torch.cuda.stream(b):
            g = torch.as_tensor(t.dataToGPU(b.cuda_stream), device="cuda")
            assert g.double().sum().item() == 50.0 * (i + 1) * n
        del g
        t.dispose()
        a.wait_stream(b)
    assert backend.numDataIds() == before


def test_what_is_pending_on_a_handed_out_tensor_saw_it_before(cuda_engine):
    """An operation that was called before its operand's memory was handed out, or while somebody has
    it, gives what it gives when launched at once."""
    from tfjs_b200 import ops as tf
    backend = cuda_engine.backend
    before = backend.numDataIds()
    stream = torch.cuda.current_stream().cuda_stream
    t = tf.tensor(np.full(10000, 3.0, np.float32))
    y = tf.add(t, t)                                    # deferred
    assert not backend.lazy_fusion or backend.pending_of(y.dataId) is not None
    g = torch.as_tensor(t.dataToGPU(stream), device="cuda")
    g.zero_()
    torch.cuda.synchronize()
    assert np.all(y.arraySync() == 6.0)
    z = tf.add(t, t)                                    # while g is there
    backend.signal_stream(stream)
    g.fill_(5.0)
    torch.cuda.synchronize()
    assert np.all(z.arraySync() == 0.0)
    backend.wait_stream(stream)
    del g
    u = tf.add(t, t)                                    # nobody else has it any more
    assert not backend.lazy_fusion or backend.pending_of(u.dataId) is not None
    assert np.all(u.arraySync() == 10.0)
    for k in (t, y, z, u):
        k.dispose()
    assert backend.numDataIds() == before


def _conv(tf, x, f):
    return tf.conv2d(x, f, 1, "same")


@pytest.mark.parametrize("size,channels", [(1, 64), (3, 32), (3, 6)])
def test_a_foreign_filter_is_read_anew(cuda_engine, size, channels):
    """A filter whose owner rewrites it: each convolution uses what is there, not a copy that an
    earlier one made; a captured one as well."""
    from tfjs_b200 import ops as tf
    backend = cuda_engine.backend
    backend.set_math_mode("tf32")
    r = np.random.default_rng(size + channels)
    x = tf.tensor(r.standard_normal((2, 14, 14, channels)).astype(np.float32))
    values = [r.standard_normal((size, size, channels, 64)).astype(np.float32) for _ in range(3)]
    own = [tf.tensor(v) for v in values]
    refs = [_conv(tf, x, f) for f in own]
    want = [t.arraySync() for t in refs]
    mem = torch.from_numpy(values[0]).cuda()
    torch.cuda.synchronize()
    f = tf.tensor(mem)
    outs = []
    for i in range(2):
        mem.copy_(torch.from_numpy(values[i]))
        torch.cuda.synchronize()
        outs.append(_conv(tf, x, f))
        assert np.array_equal(outs[-1].arraySync(), want[i])
    backend.capture_begin(16 << 20)
    out = _conv(tf, x, f)
    backend.device_id(out.dataId)
    graph = backend.capture_end()
    for i in (2, 0):
        mem.copy_(torch.from_numpy(values[i]))
        torch.cuda.synchronize()
        backend.graph_launch(graph)
        assert np.array_equal(out.arraySync(), want[i])
    backend.graph_destroy(graph)
    for t in [x, f, out] + own + refs + outs:
        t.dispose()


@pytest.mark.parametrize("product", ["matmul", "conv"])
def test_a_handed_out_weight_is_read_anew(cuda_engine, product):
    """A weight that its holder rewrites: products see it, a captured step with the old copy is
    refused, and once nobody holds it any more one copy serves again."""
    from tfjs_b200 import _cabi, ops as tf
    backend = cuda_engine.backend
    backend.set_math_mode("tf32")
    r = np.random.default_rng(5)
    if product == "matmul":
        a = tf.tensor(r.standard_normal((96, 64)).astype(np.float32))
        w = tf.tensor(r.standard_normal((64, 128)).astype(np.float32))
        f = lambda: tf.mat_mul(a, w)                                       # noqa: E731
    else:
        a = tf.tensor(r.standard_normal((2, 9, 9, 32)).astype(np.float32))
        w = tf.tensor(r.standard_normal((3, 3, 32, 64)).astype(np.float32))
        f = lambda: _conv(tf, a, w)                                        # noqa: E731

    def value():
        t = f()
        v = t.arraySync()
        t.dispose()
        return v
    first = value()
    backend.capture_begin(16 << 20)
    out = f()
    backend.device_id(out.dataId)
    graph = backend.capture_end()
    g = torch.as_tensor(w.dataToGPU(torch.cuda.current_stream().cuda_stream), device="cuda")
    with pytest.raises(_cabi.CudaError) as e:
        backend.graph_launch(graph)
    assert e.value.code == _cabi.UNSUPPORTED
    for factor in (2.0, 0.25):                        # powers of two: the products scale exactly
        g.mul_(factor)
        torch.cuda.synchronize()
        first = first * np.float32(factor)
        assert np.array_equal(value(), first)
    del g
    assert np.array_equal(value(), first)
    backend.launch_log(True)
    assert np.array_equal(value(), first)
    log = backend.launch_log_take()
    backend.launch_log(False)
    assert log and "pack_weight" not in log
    backend.graph_destroy(graph)
    for t in (a, w, out):
        t.dispose()


def test_a_holder_that_goes_away_during_a_capture(cuda_engine):
    """Neither side's capture is disturbed, and the memory is used again only behind the holder's work."""
    from tfjs_b200 import ops as tf
    backend = cuda_engine.backend
    before = backend.numDataIds()
    side = torch.cuda.Stream()
    n = 1 << 22
    x = tf.tensor(np.arange(n, dtype=np.float32))
    y = tf.tensor(np.full(5000, 2.0, np.float32))
    g = torch.as_tensor(x.dataToGPU(side.cuda_stream), device="cuda")
    x.dispose()
    with torch.cuda.stream(side):
        total = torch.zeros((), device="cuda", dtype=torch.float64)
        for _ in range(20):
            total += g.double().sum()
    backend.capture_begin(1 << 20)
    del g
    z = tf.mul(y, y)
    backend.device_id(z.dataId)
    graph = backend.capture_end()
    w = tf.tensor(np.zeros(n, np.float32))             # of the same size: may take that block
    backend.graph_launch(graph)
    assert np.all(z.arraySync() == 4.0)
    with torch.cuda.stream(side):
        assert total.item() == 20 * (float(n) * (n - 1) / 2)
    # the holder captures a graph of its own on that stream
    g = torch.as_tensor(w.dataToGPU(side.cuda_stream), device="cuda")
    w.dispose()
    torch.cuda.synchronize()
    theirs = torch.cuda.CUDAGraph()
    with torch.cuda.graph(theirs, stream=side):
        total += 1.0
        del g
    assert backend.numDataIds() == before + 3          # y, z, and what w held
    backend.sync()
    assert backend.numDataIds() == before + 2
    backend.graph_destroy(graph)
    for t in (y, z):
        t.dispose()
    assert backend.numDataIds() == before


def test_a_copy_over_a_small_tensor(cuda_engine):
    """backend.copy, which hands a captured step's results to its next replay: a small tensor written
    from the host reads as the copy left it, and what is pending on the old contents saw those."""
    from tfjs_b200 import ops as tf
    backend = cuda_engine.backend
    t, s = tf.tensor(np.array([1, 2, 3], np.int32)), tf.tensor(np.array([7, 8, 9], np.int32))
    backend.copy(s.dataId, t.dataId)
    assert list(t.arraySync()) == [7, 8, 9] and list(s.arraySync()) == [7, 8, 9]
    x, y = tf.tensor(np.full(5000, 1.0, np.float32)), tf.tensor(np.full(5000, 4.0, np.float32))
    z = tf.add(x, x)
    backend.copy(y.dataId, x.dataId)
    assert np.all(z.arraySync() == 2.0) and np.all(x.arraySync() == 4.0)
    for k in (t, s, x, y, z):
        k.dispose()


def test_a_tensor_that_its_holder_fills(cuda_engine):
    """New memory, handed out before any kernel has written it."""
    from tfjs_b200 import ops as tf
    backend = cuda_engine.backend
    before = backend.numDataIds()
    side = torch.cuda.Stream()
    for n in (1000, 1 << 23, 1 << 23, 3001):
        backend.signal_stream(side.cuda_stream)
        t = cuda_engine.make_tensor_from_info(backend.make_output([n], "float32"))
        with torch.cuda.stream(side):
            g = torch.as_tensor(t.dataToGPU(side.cuda_stream), device="cuda")
            g.copy_(torch.arange(n, device="cuda"))
        backend.wait_stream(side.cuda_stream)
        y = tf.add(t, t)
        assert np.array_equal(y.arraySync(), 2.0 * np.arange(n, dtype=np.float32))
        del g
        t.dispose()
        y.dispose()
    assert backend.numDataIds() == before
