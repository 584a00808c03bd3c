"""What the host side of the backend asks of the library when device memory changes hands, on a
stand-in for the library that records the calls."""
import pytest

from tfjs_b200 import _cabi
from tfjs_b200.backend import CudaBackend, TensorInfo


class Library(object):
    """Every call succeeds; `calls` holds their names, ids and addresses are made up, and `fail` gives
    the status of calls that are to fail."""

    def __init__(self):
        self.calls, self.fail, self.ids, self.freed = [], {}, 0, []

    def __getattr__(self, name):
        if not name.startswith("tfjs_cuda_"):
            raise AttributeError(name)
        name = name[len("tfjs_cuda_"):]

        def call(*args):
            self.calls.append(name)
            if name == "last_error":
                return b"made to fail"
            if name in self.fail:
                return self.fail[name]
            if name in ("alloc", "upload", "from_device"):
                self.ids += 1
                args[-1]._obj.value = self.ids
            elif name == "device_ptr":
                args[-1]._obj.value = 4096 * args[1]
            elif name == "create":
                args[-1]._obj.value = 1
            elif name == "capture_end":
                args[-1]._obj.value = 1
            elif name == "free":
                self.freed.append(args[1])
            return 0
        return call

    def taken(self):
        calls, self.calls = self.calls, []
        return calls


class Deferred(object):
    """A deferred kernel over `reads`."""

    def __init__(self, *reads, fails=False):
        self.reads, self.fails, self.desc = reads, fails, None

    def deps(self):
        return list(self.reads)

    def launch(self, backend, dev, post_act):
        backend.lib.tfjs_cuda_a_kernel(backend.ctx)
        if self.fails:
            raise RuntimeError("a launch that fails")


class Memory(object):
    """Another library's."""

    def __init__(self, shape=(2000,), read_only=False, **more):
        self.__cuda_array_interface__ = dict({"shape": shape, "typestr": "<f4", "strides": None,
                                              "data": (1 << 20, read_only), "version": 3}, **more)


@pytest.fixture
def backend(monkeypatch):
    lib = Library()
    monkeypatch.setattr(_cabi, "load", lambda: lib)
    b = CudaBackend(0)
    lib.taken()
    yield b
    b.ctx = None


def test_handing_out_takes_a_reference(backend):
    """The caller's handle is the caller's: of a TensorInfo and of an engine's tensor."""
    from tfjs_b200.engine import Engine
    t = backend.make_output([2000], "float32")
    g = backend.readToGPU(t, 7)
    assert g.buffer == 4096 * backend.data[t.dataId].dev and g.bufSize == 8000
    g.dispose()
    g.dispose()
    assert backend.refCount(t.dataId) == 1 and backend.lib.freed == []
    g = backend.readToGPU(t)
    backend.disposeData(t.dataId)
    assert backend.lib.freed == []
    g.dispose()
    assert len(backend.lib.freed) == 1 and backend.numDataIds() == 0
    engine = Engine()
    engine.backend = backend
    x = engine.make_tensor_from_info(backend.make_output([2000], "float32"))
    g = backend.readToGPU(x)
    h = x.dataToGPU(7)
    del g, h
    assert not x.isDisposed and backend.refCount(x.dataId) == 1
    backend.lib.fail["device_ptr"] = 2
    for f in (backend.readToGPU, lambda y: y.dataToGPU()):
        with pytest.raises(_cabi.CudaError):
            f(x)
    assert backend.refCount(x.dataId) == 1
    x.dispose()
    assert backend.numDataIds() == 0 and engine.num_tensors == 0


def test_readers_launch_before_an_address_is_handed_out(backend):
    t = backend.make_output([2000], "float32")
    y = backend.defer([2000], "float32", Deferred(t.dataId))
    backend.lib.taken()
    g = backend.readToGPU(t, 7)
    assert backend.lib.taken() == ["alloc", "a_kernel", "device_ptr", "signal_stream"]
    assert backend.pending_of(y.dataId) is None
    # while somebody holds it, what reads it launches at once
    z = backend.defer([2000], "float32", Deferred(t.dataId))
    assert backend.lib.taken() == ["alloc", "a_kernel"] and backend.pending_of(z.dataId) is None
    g2 = backend.readToGPU(t, 7)
    g.dispose()
    assert backend.pending_of(backend.defer([2000], "float32", Deferred(t.dataId)).dataId) is None
    g2.dispose()
    assert backend.pending_of(backend.defer([2000], "float32", Deferred(y.dataId)).dataId) is not None


def test_the_library_is_told_when_nobody_holds_a_tensor_any_more(backend):
    t = backend.make_output([2000], "float32")
    g, g2 = backend.readToGPU(t, 7), backend.readToGPU(t)
    backend.lib.taken()
    g.dispose()
    assert backend.lib.taken() == ["wait_stream", "device_ptr_end"]
    backend.disposeData(t.dataId)
    g2.dispose()
    assert backend.lib.taken() == ["free"]
    t = backend.make_output([2000], "float32")
    backend.lib.fail["signal_stream"] = 2
    backend.lib.taken()
    with pytest.raises(_cabi.CudaError):
        backend.readToGPU(t, 7)
    assert backend.lib.taken() == ["device_ptr", "signal_stream", "last_error", "device_ptr_end"]


def test_memory_is_kept_until_its_holders_stream_can_be_waited_for(backend):
    """Not freed in front of the holder's work: not during a capture, which the wait would discard, and
    not while the holder's own stream is being captured."""
    t, u = backend.make_output([2000], "float32"), backend.make_output([2000], "float32")
    held = [backend.readToGPU(x, 7) for x in (t, u)]
    for x in (t, u):
        backend.disposeData(x.dataId)
    backend.capture_begin(1 << 20)
    backend.lib.taken()
    held.pop().dispose()
    assert backend.lib.taken() == [] and backend.lib.freed == []
    backend.capture_end()
    assert backend.lib.taken() == ["capture_end", "wait_stream", "free"]
    backend.lib.fail["wait_stream"] = _cabi.UNSUPPORTED
    held.pop().dispose()
    assert len(backend.lib.freed) == 1
    del backend.lib.fail["wait_stream"]
    backend.lib.taken()
    backend.sync()
    assert backend.lib.taken() == ["wait_stream", "free", "sync"] and backend.numDataIds() == 0
    # a capture that ends badly, and one that never began
    v = backend.make_output([2000], "float32")
    g = backend.readToGPU(v, 7)
    backend.disposeData(v.dataId)
    backend.capture_begin(1 << 20)
    g.dispose()
    backend.lib.fail["capture_end"] = 2
    with pytest.raises(_cabi.CudaError):
        backend.capture_end()
    assert backend.numDataIds() == 0
    backend.lib.fail["capture_begin"] = 2
    with pytest.raises(_cabi.CudaError):
        backend.capture_begin(1 << 20)
    w = backend.make_output([2000], "float32")
    g = backend.readToGPU(w, 7)
    backend.disposeData(w.dataId)
    g.dispose()
    assert backend.numDataIds() == 0


def test_foreign_memory_is_referenced_until_its_owners_stream_can_be_signalled(backend):
    import sys
    memory = Memory()
    count = sys.getrefcount(memory)
    t = backend.createTensorFromGPUData(memory, stream=7)
    backend.lib.fail["signal_stream"] = _cabi.UNSUPPORTED       # (its owner captures a graph there)
    backend.disposeData(t.dataId)
    assert backend.numDataIds() == 0 and sys.getrefcount(memory) > count
    backend.sync()
    assert sys.getrefcount(memory) > count
    del backend.lib.fail["signal_stream"]
    backend.lib.taken()
    backend.sync()
    assert backend.lib.taken() == ["signal_stream", "sync"] and sys.getrefcount(memory) == count


def test_read_only_memory_and_the_interfaces_own_stream(backend):
    from tfjs_b200.kernels import decoder
    waited = []
    plain = backend.lib.tfjs_cuda_wait_stream
    backend.lib.tfjs_cuda_wait_stream = lambda ctx, stream: waited.append(stream) or plain(ctx, stream)
    pool = [9, 2, 16, 64]
    kc = backend.createTensorFromGPUData(Memory(pool, read_only=True, stream=5))
    assert waited == [5]
    vc = backend.createTensorFromGPUData(Memory(pool, stream=None))
    backend.createTensorFromGPUData(Memory(pool, stream=1), stream=9)
    assert waited == [5, 9]
    make = lambda shape, dtype="float32": backend.make_output(shape, dtype)     # noqa: E731
    inp = {"kCache": kc, "vCache": vc, "pageTable": make([3, 4], "int32"), "lengths": make([3], "int32"),
           "k": make([3, 2, 1, 64]), "v": make([3, 2, 1, 64]), "weights": make([3, 2, 64])}
    backend.lib.taken()
    for kernel, attrs in ((decoder._paged_cache_append, {}), (decoder._paged_cache_evict, {"budget": 8})):
        for names in (("kCache", "vCache"), ("vCache", "kCache")):
            pools = dict(zip(names, (kc, vc)))
            with pytest.raises(ValueError, match="read-only"):
                kernel({"backend": backend, "inputs": dict(inp, **pools), "attrs": attrs})
    assert not [c for c in backend.lib.taken() if c.startswith("paged")]
    inp["q"] = make([3, 4, 1, 64])
    decoder._paged_attention({"backend": backend, "inputs": dict(inp, weights=None), "attrs": {}})
    g, h = backend.readToGPU(kc), backend.readToGPU(vc)
    assert g.__cuda_array_interface__["data"][1] is True and h.__cuda_array_interface__["data"][1] is False


def test_a_copy_writes_its_destination(backend):
    import numpy as np
    src, dst = backend.make_output([2], "float32"), TensorInfo(backend.write(np.zeros(2), [2], "float32"), [2], "float32")
    y = backend.defer([2], "float32", Deferred(dst.dataId))
    backend.lib.taken()
    backend.copy(src.dataId, dst.dataId)
    assert backend.lib.taken() == ["alloc", "a_kernel", "alloc", "write", "copy"]
    assert backend.pending_of(y.dataId) is None and backend.host_values(dst.dataId) is None
    backend.copy(src.dataId, src.dataId)
    locked = backend.createTensorFromGPUData(Memory((2,), read_only=True))
    with pytest.raises(ValueError, match="read-only"):
        backend.copy(src.dataId, locked.dataId)


def test_two_threads_get_their_own_ids(backend):
    """The library's calls let other threads run: each caller's new id is its own."""
    import threading
    inside, go_on = threading.Event(), threading.Event()
    plain, first = backend.lib.tfjs_cuda_alloc, []

    def alloc(ctx, nbytes, out):
        rc = plain(ctx, nbytes, out)
        if not first:
            first.append(out._obj.value)
            inside.set()
            go_on.wait(10)
        return rc
    backend.lib.tfjs_cuda_alloc = alloc
    made = []
    other = threading.Thread(target=lambda: made.append(backend.make_output([2000], "float32")))
    other.start()
    assert inside.wait(10)
    mine = backend.make_output([2000], "float32")
    foreign = backend.createTensorFromGPUData(Memory())
    go_on.set()
    other.join(10)
    ids = [backend.data[t.dataId].dev for t in (made[0], mine, foreign)]
    assert ids == [1, 2, 3]


def test_a_launch_that_fails_leaves_nothing_behind(backend):
    t = backend.createTensorFromGPUData(Memory())
    u = backend.make_output([2000], "float32")
    with pytest.raises(RuntimeError):
        backend.defer([2000], "float32", Deferred(t.dataId, u.dataId, fails=True))
    assert backend.numDataIds() == 2 and backend.refCount(t.dataId) == backend.refCount(u.dataId) == 1
    assert backend.data[t.dataId].held == 0
    for x in (t, u):
        assert backend.disposeData(x.dataId)
    assert len(backend.data) == 0 and len(backend.lib.freed) == 3


def test_a_tensors_info_is_the_callers(backend):
    """A kernel that changes what it was given does not change the tensor, nor one that shares its data."""
    from tfjs_b200.engine import Engine
    engine = Engine()
    engine.backend = backend
    x = engine.make_tensor_from_info(backend.make_output([20, 100], "float32"))
    first = x.info()
    first.dtype = "int32"
    again = x.info()
    assert (again.shape, again.dtype, again.dataId) == ([20, 100], "float32", x.dataId)
    assert x.shape == [20, 100] and x.dtype == "float32"
    x.dispose()


def test_masked_memory_is_refused(backend):
    with pytest.raises(ValueError, match="mask"):
        backend.createTensorFromGPUData(Memory(mask=Memory()))
    assert backend.numDataIds() == 0 and backend.lib.taken() == []
    backend.createTensorFromGPUData(Memory(mask=None))
