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
