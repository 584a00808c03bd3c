"""Tensors over another library's device memory (createTensorFromGPUData) and the way back
(dataToGPU), without copies and in order with the other library's stream."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def test_a_tensor_over_foreign_memory(cuda_engine):
    from tfjs_b200 import ops as tf
    backend = cuda_engine.backend
    before, used = backend.numDataIds(), backend.memory()["numBytesInGPU"]
    x = torch.randn(5, 33, device="cuda")
    torch.cuda.synchronize()
    t = tf.tensor(x)
    assert t.shape == [5, 33] and t.dtype == "float32"
    assert backend.memory()["numBytesInGPU"] == used
    assert np.array_equal(t.arraySync(), x.cpu().numpy())
    x.mul_(2.0)
    torch.cuda.synchronize()
    assert np.array_equal(t.arraySync(), x.cpu().numpy())       # the same memory
    y = tf.add(t, t)
    assert np.array_equal(y.arraySync(), x.cpu().numpy() * 2)
    i = tf.tensor(torch.arange(7, dtype=torch.int32, device="cuda"), shape=[7, 1])
    assert i.dtype == "int32" and i.shape == [7, 1]
    for k in (t, y, i):
        k.dispose()
    assert backend.numDataIds() == before and np.isfinite(x.sum().item())


def test_there_and_back_on_a_stream(cuda_engine):
    """Producer on a side stream, this backend, consumer on the side stream: no host wait in
    between; the consumer's memory outlives the tensor's handle."""
    from tfjs_b200 import ops as tf
    backend = cuda_engine.backend
    before = backend.numDataIds()
    side = torch.cuda.Stream()
    for n in (1000, 1 << 24):
        with torch.cuda.stream(side):
            x = torch.zeros(n, device="cuda")
            for _ in range(20):
                x += 1.0
            t = tf.tensor(x, stream=side.cuda_stream)
            y = tf.mul(t, t)
            t.dispose()
            x.zero_()                       # behind the product, which read it
            g = torch.as_tensor(y.dataToGPU(side.cuda_stream), device="cuda")
            y.dispose()
            total, rest = g.double().sum().item(), x.sum().item()     # (read on the side stream)
        assert total == 400.0 * n
        assert rest == 0.0
        del g
    assert backend.numDataIds() == before


def test_what_reads_foreign_memory_launches_at_once(cuda_engine):
    """Elementwise kernels are usually deferred; over memory that its owner may rewrite they are not."""
    from tfjs_b200 import ops as tf
    stream = torch.cuda.current_stream().cuda_stream
    x = torch.ones(10000, device="cuda")
    t = tf.tensor(x, stream=stream)
    y = tf.add(t, t)
    cuda_engine.backend.signal_stream(stream)
    x.fill_(7.0)
    z = tf.mul(y, y)
    assert np.all(z.arraySync() == 4.0)
    for k in (t, y, z):
        k.dispose()
    # the tensor is forgotten even where the stream cannot be signalled: inside a captured step
    before = cuda_engine.backend.numDataIds()
    t = tf.tensor(x, stream=stream)
    cuda_engine.backend.capture_begin(1 << 20)
    with pytest.raises(Exception):
        t.dispose()
    with pytest.raises(Exception):
        cuda_engine.backend.capture_end()
    assert cuda_engine.backend.numDataIds() == before
    assert np.all(x.cpu().numpy() == 7.0)


def test_a_host_resident_tensor_goes_to_the_gpu(cuda_engine):
    from tfjs_b200 import ops as tf
    t = tf.tensor(np.arange(6, dtype=np.float32).reshape(2, 3))
    stream = torch.cuda.current_stream().cuda_stream
    g = torch.as_tensor(t.dataToGPU(stream), device="cuda")
    g += 1.0
    torch.cuda.synchronize()
    assert np.array_equal(t.arraySync(), np.arange(6).reshape(2, 3) + 1.0)
    del g
    t.dispose()


def test_refusals(cuda_engine):
    from tfjs_b200 import ops as tf, _cabi
    backend = cuda_engine.backend
    before = backend.numDataIds()
    with pytest.raises(ValueError):
        tf.tensor(torch.zeros(4, 4, device="cuda").t()[1:])
    with pytest.raises(ValueError):
        tf.tensor(torch.zeros(4, device="cuda", dtype=torch.float16))

    class At(object):
        def __init__(self, ptr):
            self.__cuda_array_interface__ = {"shape": (4,), "typestr": "<f4", "strides": None,
                                             "data": (ptr, False), "version": 2}
    x = torch.zeros(64, device="cuda")
    host = torch.zeros(64)
    for ptr in (x.data_ptr() + 4, host.data_ptr() // 16 * 16 + 16, 0):
        with pytest.raises(_cabi.CudaError) as e:
            tf.tensor(At(ptr))
        assert e.value.code == 1
    assert backend.numDataIds() == before
    # neither order nor memory of others inside a captured step
    backend.sync()
    backend.capture_begin(1 << 20)
    with pytest.raises(_cabi.CudaError) as e:
        backend.wait_stream(0)
    assert e.value.code == _cabi.UNSUPPORTED
    with pytest.raises(_cabi.CudaError):
        backend.capture_end()
    backend.sync()
