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
